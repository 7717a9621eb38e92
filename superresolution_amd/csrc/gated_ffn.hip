// Host entry points of the gated feed-forward block (srmi_gated_ffn, srmi_gated_ffn_backward); the kernels are in
// gated_ffn_kernel.h.
#include "gated_ffn.h"

namespace srmi {

constexpr int kFfnMaxC = 4096, kFfnMaxHidden = 16384;
// Hidden tensors of one run of pixels in the workspace.  Few long runs beat runs that stay in the 256 MiB Infinity Cache: each run of
// the backward pass adds a row of the weights' partial sums per split (131072 pixels, c 256, hidden 1024: one run 823 us, four 1005).
constexpr long long kFfnRunBytes = 4ll << 30;
constexpr unsigned kFfnTile = 256;   // pixels of a workgroup of the tile kernels

static const FfnLaunch* ffn_table(int dtype) { return dtype == SRMI_F16 ? srmi_ffn_f16() : dtype == SRMI_BF16 ? srmi_ffn_bf16() : srmi_ffn_f32(); }

static bool ffn_shape_ok(int dtype, int n, int h, int w, int c, int hidden) {
    if (dtype != SRMI_F32 && dtype != SRMI_F16 && dtype != SRMI_BF16) return false;
    const int cpb = dtype_cpb(dtype);
    return n > 0 && h > 0 && w > 0 && c > 0 && hidden > 0 && c % cpb == 0 && hidden % cpb == 0 && c <= kFfnMaxC && hidden <= kFfnMaxHidden &&
           (long long)n * h * w < (1ll << 31);
}

static int ffn_check(const char* who, int dtype, int n, int h, int w, int c, int hidden, int act) {
    if (dtype != SRMI_F32 && dtype != SRMI_F16 && dtype != SRMI_BF16) SRMI_FAIL("%s: the compute type must be f32, f16 or bf16", who);
    if (!ffn_shape_ok(dtype, n, h, w, c, hidden))
        SRMI_FAIL("%s: bad shape n=%d h=%d w=%d c=%d hidden=%d (c and hidden: multiples of the plane width %d, at most %d and %d; fewer than 2^31 pixels)", who, n,
                  h, w, c, hidden, dtype_cpb(dtype), kFfnMaxC, kFfnMaxHidden);
    if (act < SRMI_ACT_NONE || act > SRMI_ACT_GELU) SRMI_FAIL("%s: bad activation %d", who, act);
    return 0;
}

static int ffn_check_tensor(const char* who, const char* name, const srmi_tensor_t& t, int dtype, bool may_miss) {
    if (!t.ptr) {
        if (may_miss) return 0;
        SRMI_FAIL("%s: no %s", who, name);
    }
    if (t.dtype != dtype) SRMI_FAIL("%s: %s must be of the compute type", who, name);
    const long long es = dtype_size(dtype);
    if (((uintptr_t)t.ptr | (unsigned long long)(t.img_stride * es) | (unsigned long long)(t.plane_stride * es)) & 15)
        SRMI_FAIL("%s: address and strides of %s must be multiples of 16 bytes", who, name);
    return 0;
}

static int ffn_check_weights(const char* who, const void* a, const void* b, const void* c) {
    if (!a || !b || !c) SRMI_FAIL("%s: null weight", who);
    if (((uintptr_t)a | (uintptr_t)b | (uintptr_t)c) & 15) SRMI_FAIL("%s: weights must lie on multiples of 16 bytes", who);
    return 0;
}

static FfnParams ffn_params(int dtype, int n, int h, int w, int c, int hidden, float res_scale) {
    FfnParams p = {};
    p.hw = (unsigned)h * (unsigned)w;
    p.m = (unsigned)n * p.hw;
    unsigned l = 0;
    while (l < 31 && (1u << l) < p.hw) ++l;
    p.hw_shift = l;
    p.hw_mul = (unsigned)((((1ull << l) - p.hw) << 32) / p.hw + 1);
    p.c = c;
    p.hidden = hidden;
    p.kp_c = c / dtype_cpb(dtype);
    p.kp_h = hidden / dtype_cpb(dtype);
    p.res_scale = res_scale;
    return p;
}

// Pixels of a launch: all of them, or runs of equal length whose `tensors` hidden tensors fit kFfnRunBytes
static unsigned ffn_run_pixels(unsigned m, int kp_h, int tensors) {
    const long long most = kFfnRunBytes / ((long long)kp_h * 32 * tensors);
    const unsigned cap = most < kFfnTile ? kFfnTile : (unsigned)(most < (1ll << 30) ? most : (1ll << 30)) / kFfnTile * kFfnTile;
    const unsigned runs = (m + cap - 1) / cap;
    const unsigned per = ((m + runs - 1) / runs + kFfnTile - 1) / kFfnTile * kFfnTile;
    return per < m ? per : m;
}

static size_t ffn_hidden_bytes(unsigned run, int kp_h) {
    return (size_t)((run + kFfnHiddenBlock - 1) / kFfnHiddenBlock) * kFfnHiddenBlock * 32 * kp_h;
}

// Parts of the hidden units (chunks of 32) that the one-launch form runs side by side: as many as bring the launch to half a
// workgroup per CU.  Going on to a whole one adds more f32 partial sums than it takes off the walk.
static unsigned ffn_parts(int dtype, unsigned m, int c, int hidden) {
    const unsigned px = c / dtype_cpb(dtype) > 12 ? 256 : 128, tiles = (m + px - 1) / px, chunks = (hidden + 31) / 32;
    const unsigned want = 128 / tiles;
    return want < 2 ? 1 : want < chunks ? want : chunks;
}

// The backward pass's workspace
struct FfnPlan {
    unsigned run, runs;        // pixels of a run
    unsigned split, splits;    // pixels of a split of the weight gradients' sums, splits of a run
    unsigned tile, tiles;      // pixels of a workgroup that leaves bias sums, workgroups of all runs
    unsigned fold;             // rows of the bias sums that a launch before the last adds (0: none)
    unsigned parts, dx_parts;  // parts of the hidden units in the launch that walks them, partial sums of dx
    size_t hid, dx_part, transposed, wpart, bias_part, bias_fold, db_part, total;
};
static FfnPlan ffn_plan(int dtype, unsigned m, int c, int hidden, bool bias_hidden, bool bias_down) {
    FfnPlan q = {};
    const int kp_h = hidden / dtype_cpb(dtype), es = dtype_size(dtype);
    q.run = ffn_run_pixels(m, kp_h, 3);
    q.runs = (m + q.run - 1) / q.run;
    const int cols = ffn_wgrad_cols(c), kp_c = c / dtype_cpb(dtype);
    const unsigned wtiles = 3u * ((c + cols - 1) / cols) * ((hidden + 255) / 256);
    // One workgroup per CU, but not for fewer than 128 pixels, since every split adds a row of partial sums (f32, 4096 pixels, c 256,
    // hidden 512: 171 us with at least 256, 145 with 128 or 64; f16, 2000 pixels, c 128, hidden 256: 30.7, 30.0 and 32.5).
    const unsigned want = wtiles < 256 ? 256 / wtiles : 1;
    q.split = ((q.run + want - 1) / want + 63) / 64 * 64;
    if (q.split < 128) q.split = 128;
    q.splits = (q.run + q.split - 1) / q.split;
    q.tile = kp_c <= kFfnBackPlanes ? kFfnBackTile : kp_c <= kFfnFusedPlanes ? kFfnBackTileWide : kFfnTile;
    q.tiles = q.runs * ((q.run + q.tile - 1) / q.tile);
    // one workgroup per CU.  dx's partial sums are joined once, so they are left for one run only (where there are more, each
    // has pixels enough unless the hidden units are in the ten thousands).
    const unsigned chunks = (hidden + 31) / 32, fill = 256 / ((q.run + q.tile - 1) / q.tile);
    q.parts = kp_c > kFfnFusedPlanes || fill < 2 || (q.runs > 1 && kp_c <= kFfnBackPlanes) ? 1 : fill < chunks ? fill : chunks;
    q.dx_parts = q.runs > 1 ? 1 : kp_c <= kFfnBackPlanes ? q.parts : ffn_tile_parts(m, c, kp_h, false);
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t r = at; at += (bytes + 255) & ~(size_t)255; return r; };
    q.hid = take(3 * ffn_hidden_bytes(q.run, kp_h));
    q.dx_part = take(q.dx_parts > 1 ? (size_t)q.dx_parts * q.run * c * sizeof(float) : 0);
    q.transposed = take(kp_c > kFfnBackPlanes ? (size_t)3 * c * hidden * es : 0);
    q.wpart = take((size_t)q.runs * q.splits * 3 * c * hidden * sizeof(float));
    q.bias_part = take(bias_hidden ? (size_t)q.tiles * 2 * hidden * sizeof(float) : 0);
    q.fold = bias_hidden ? ffn_bias_fold(q.tiles) : 0;
    q.bias_fold = take(q.fold ? (size_t)((q.tiles + q.fold - 1) / q.fold) * 2 * hidden * sizeof(float) : 0);
    q.db_part = take(bias_down ? (size_t)q.runs * q.splits * ffn_wgrad_bias_rows(c) * c * sizeof(float) : 0);
    q.total = at;
    return q;
}

}  // namespace srmi

using namespace srmi;

extern "C" size_t srmi_gated_ffn_workspace(const srmi_gated_ffn_desc_t* d) {
    if (!d || !ffn_shape_ok(d->dtype, d->n, d->h, d->w, d->c, d->hidden)) return 0;
    const int cpb = dtype_cpb(d->dtype), kp_h = d->hidden / cpb;
    const unsigned m = (unsigned)d->n * d->h * d->w;
    if (d->c / cpb <= kFfnFusedPlanes) {
        const unsigned parts = ffn_parts(d->dtype, m, d->c, d->hidden);
        return parts > 1 ? (size_t)parts * m * d->c * sizeof(float) : 0;
    }
    const unsigned run = ffn_run_pixels(m, kp_h, 1), parts = run < m ? 1 : ffn_tile_parts(m, d->c, kp_h, true);
    return ffn_hidden_bytes(run, kp_h) + (parts > 1 ? (size_t)parts * m * d->c * sizeof(float) : 0);
}

extern "C" int srmi_gated_ffn(const srmi_gated_ffn_desc_t* d, void* workspace, size_t workspace_bytes, void* hip_stream) {
    const char* who = "srmi_gated_ffn";
    if (!d) SRMI_FAIL("%s: null descriptor", who);
    if (ffn_check(who, d->dtype, d->n, d->h, d->w, d->c, d->hidden, d->act) || ffn_check_tensor(who, "x", d->x, d->dtype, false) ||
        ffn_check_tensor(who, "res", d->res, d->dtype, true) || ffn_check_tensor(who, "out", d->out, d->dtype, false) ||
        ffn_check_weights(who, d->w_gate, d->w_up, d->w_down))
        return -1;
    if (d->x.ptr == d->out.ptr) SRMI_FAIL("%s: out must not be x", who);
    const size_t need = srmi_gated_ffn_workspace(d);
    if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15)))
        SRMI_FAIL("%s: needs %zu bytes of workspace on a multiple of 16 (got %zu)", who, need, workspace ? workspace_bytes : (size_t)0);
    FfnParams p = ffn_params(d->dtype, d->n, d->h, d->w, d->c, d->hidden, d->res_scale);
    p.x = to_view(d->x); p.res = to_view(d->res); p.out = to_view(d->out);
    p.w_gate = (const char*)d->w_gate; p.w_up = (const char*)d->w_up; p.w_down = (const char*)d->w_down;
    p.b_gate = d->b_gate; p.b_up = d->b_up; p.b_down = d->b_down;
    p.hid = (char*)workspace;
    const FfnLaunch* f = ffn_table(d->dtype);
    hipStream_t s = (hipStream_t)hip_stream;
    if (p.kp_c <= kFfnFusedPlanes) {
        const unsigned parts = ffn_parts(d->dtype, p.m, p.c, p.hidden);
        p.part = parts > 1 ? (float*)workspace : nullptr;
        if (f->fused(p, parts, d->act, s)) return -1;
        return parts > 1 ? f->join(p, (int)parts, s) : 0;
    }
    const unsigned m = p.m, run = ffn_run_pixels(m, p.kp_h, 1);
    p.parts = run < m ? 1 : ffn_tile_parts(m, p.c, p.kp_h, true);
    p.part = p.parts > 1 ? (float*)((char*)workspace + ffn_hidden_bytes(run, p.kp_h)) : nullptr;
    for (unsigned m0 = 0; m0 < m; m0 += run) {
        p.m0 = m0;
        p.m = m - m0 < run ? m : m0 + run;
        if (f->gemm(p, kFfnHidden, d->act, s) || f->gemm(p, kFfnDown, d->act, s)) return -1;
    }
    return p.parts > 1 ? f->join(p, (int)p.parts, s) : 0;
}

extern "C" size_t srmi_gated_ffn_backward_workspace(const srmi_gated_ffn_grad_desc_t* d) {
    if (!d || !ffn_shape_ok(d->dtype, d->n, d->h, d->w, d->c, d->hidden)) return 0;
    return ffn_plan(d->dtype, (unsigned)d->n * d->h * d->w, d->c, d->hidden, d->b_gate || d->b_up, d->b_down != nullptr).total;
}

extern "C" int srmi_gated_ffn_backward(const srmi_gated_ffn_grad_desc_t* d, void* workspace, size_t workspace_bytes, void* hip_stream) {
    const char* who = "srmi_gated_ffn_backward";
    if (!d) SRMI_FAIL("%s: null descriptor", who);
    if (ffn_check(who, d->dtype, d->n, d->h, d->w, d->c, d->hidden, d->act) || ffn_check_tensor(who, "x", d->x, d->dtype, false) ||
        ffn_check_tensor(who, "d_out", d->d_out, d->dtype, false) || ffn_check_tensor(who, "dx", d->dx, d->dtype, false) ||
        ffn_check_weights(who, d->w_gate, d->w_up, d->w_down) || ffn_check_weights(who, d->d_w_gate, d->d_w_up, d->d_w_down))
        return -1;
    if (d->dx.ptr == d->x.ptr || d->dx.ptr == d->d_out.ptr) SRMI_FAIL("%s: dx must not be x or d_out", who);
    if ((d->b_gate != nullptr) != (d->d_b_gate != nullptr) || (d->b_up != nullptr) != (d->d_b_up != nullptr) ||
        (d->b_down != nullptr) != (d->d_b_down != nullptr))
        SRMI_FAIL("%s: every bias comes with its gradient's place, and none without", who);
    const size_t need = srmi_gated_ffn_backward_workspace(d);
    if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15))
        SRMI_FAIL("%s: needs %zu bytes of workspace on a multiple of 16 (got %zu)", who, need, workspace ? workspace_bytes : (size_t)0);
    FfnParams p = ffn_params(d->dtype, d->n, d->h, d->w, d->c, d->hidden, d->res_scale);
    const unsigned m = p.m;
    const bool bias_hidden = d->b_gate || d->b_up;
    const FfnPlan q = ffn_plan(d->dtype, m, d->c, d->hidden, bias_hidden, d->b_down != nullptr);
    char* ws = (char*)workspace;
    p.x = to_view(d->x); p.dy = to_view(d->d_out); p.out = to_view(d->dx);
    p.w_gate = (const char*)d->w_gate; p.w_up = (const char*)d->w_up; p.w_down = (const char*)d->w_down;
    p.b_gate = d->b_gate; p.b_up = d->b_up; p.b_down = d->b_down;
    const size_t matrix = (size_t)d->c * d->hidden * dtype_size(d->dtype), hidden_bytes = ffn_hidden_bytes(q.run, p.kp_h);
    p.wt_gate = ws + q.transposed; p.wt_up = p.wt_gate + matrix; p.wt_down = p.wt_up + matrix;
    p.hid = ws + q.hid; p.dg = p.hid + hidden_bytes; p.du = p.dg + hidden_bytes;
    const FfnLaunch* f = ffn_table(d->dtype);
    hipStream_t s = (hipStream_t)hip_stream;
    if (p.kp_c > kFfnBackPlanes && f->transpose(p, s)) return -1;
    unsigned rows = 0, tiles = 0;
    for (unsigned m0 = 0; m0 < m; m0 += q.run) {
        p.m0 = m0;
        p.m = m - m0 < q.run ? m : m0 + q.run;
        p.bias_part = bias_hidden ? (float*)(ws + q.bias_part) + (size_t)tiles * 2 * p.hidden : nullptr;
        p.wpart = (float*)(ws + q.wpart) + (size_t)rows * 3 * p.c * p.hidden;
        p.db_part = d->b_down ? (float*)(ws + q.db_part) + (size_t)rows * ffn_wgrad_bias_rows(p.c) * p.c : nullptr;
        p.split_pixels = q.split;
        p.parts = q.dx_parts;
        p.part = q.dx_parts > 1 ? (float*)(ws + q.dx_part) : nullptr;
        const unsigned splits = (p.m - m0 + q.split - 1) / q.split;
        if (p.kp_c <= kFfnFusedPlanes ? f->back(p, q.parts, d->act, s) : f->gemm(p, kFfnHiddenGrad, d->act, s)) return -1;
        if (p.kp_c > kFfnBackPlanes && f->gemm(p, kFfnInputGrad, d->act, s)) return -1;
        if (f->wgrad(p, splits, s)) return -1;
        rows += splits;
        tiles += (p.m - m0 + q.tile - 1) / q.tile;
    }
    FfnFinish e = {};
    e.wpart = (const float*)(ws + q.wpart); e.bias_part = (const float*)(ws + q.bias_part); e.db_part = (const float*)(ws + q.db_part);
    e.each = (long long)p.hidden * p.c; e.hidden = p.hidden; e.c = p.c;
    e.splits = (int)rows;
    e.db_rows = (int)rows * ffn_wgrad_bias_rows(p.c);
    e.bias_rows = (int)tiles;
    e.fold = (int)q.fold;
    e.bias_fold = (float*)(ws + q.bias_fold);
    e.res_scale = d->res_scale;
    e.g_gate = d->d_w_gate; e.g_up = d->d_w_up; e.g_down = d->d_w_down;
    e.part = p.part; e.parts = (int)q.dx_parts; e.kp_c = p.kp_c; e.dx = p.out;
    e.m = p.m; e.hw = p.hw; e.hw_mul = p.hw_mul; e.hw_shift = p.hw_shift;
    e.db_gate = d->d_b_gate; e.db_up = d->d_b_up; e.db_down = d->d_b_down;
    return f->finish(e, s);
}
