// What the gated feed-forward block's host code (gated_ffn.hip) and its kernels (gated_ffn_kernel.h, one translation unit per
// compute type) share.
#pragma once
#include "common.h"

namespace srmi {

constexpr int kFfnHiddenBlock = 64;

struct FfnParams {
    unsigned m0, m;                   // first pixel of this launch and one past its last
    unsigned hw, hw_mul, hw_shift;
    int c, hidden;
    int kp_c, kp_h;                   // planes of c and of hidden
    float res_scale;
    TView x, res, out;                // forward; backward: x, dx in out
    TView dy;
    const char *w_gate, *w_up, *w_down;        // row-major weights
    const char *wt_gate, *wt_up, *wt_down;     // their transposes (backward)
    const float *b_gate, *b_up, *b_down;
    char *hid, *dg, *du;              // hidden tensors of the launch's pixels, in blocks of kFfnHiddenBlock pixels
    float* part;                      // [hidden part][plane][pixel][channel]: partial outputs (null: the launch writes out)
    unsigned parts;                   // of the tile kernels' products with c rows
    float* bias_part;                 // [pixel tile][2][hidden]
    // weight gradients
    float* wpart;                     // [split][3 * hidden * c]
    float* db_part;                   // [split][ffn_wgrad_bias_rows][c]: sums of dy
    unsigned split_pixels;
};

// What a launch of the block's tile kernel computes
enum {
    kFfnHidden = 0,      // hid = act(w_gate x + b_gate) * (w_up x + b_up)
    kFfnDown = 1,        // out = res + res_scale * (w_down hid + b_down)
    kFfnHiddenGrad = 2,  // hid, dg, du from x and dy
    kFfnInputGrad = 3    // out = wt_gate dg + wt_up du
};

// Partial sums of the gradients of weights and biases, and where the gradients go
struct FfnFinish {
    const float *wpart, *bias_part, *db_part;
    float* bias_fold;        // where sums of `fold` rows of bias_part go (0: they are few enough to be added at once)
    long long each;          // hidden * c
    int hidden, c;
    int splits, bias_rows, db_rows, fold;
    float res_scale;         // of w_down and b_down (dg and du have theirs already)
    void *g_gate, *g_up, *g_down;
    float *db_gate, *db_up, *db_down;
    unsigned w_blocks, h_blocks, b_blocks, p_blocks;  // blocks of the weights, of a hidden bias, of all biases, of a plane of dx
    // the gradient of x where parts of the hidden units left partial sums [part][plane][pixel][channel] of it
    const float* part;       // null: it is there already
    int parts, kp_c;
    TView dx;
    unsigned m, hw, hw_mul, hw_shift;
};

// Channels of a workgroup of the weight gradients' kernel: the narrowest instance that takes all, or 256 at a time
constexpr int kFfnWgradWaves = 2;  // 4 waves along hidden units, times this along channels or, up to 128 channels, along pixels
static inline int ffn_wgrad_bias_rows(int c) { return c <= 128 ? 4 * kFfnWgradWaves : 4; }  // rows of dy's sums of a split
static inline int ffn_wgrad_cols(int c) { return c <= 32 ? 32 : c <= 64 ? 64 : c <= 96 ? 96 : c <= 128 ? 128 : c <= 192 ? 192 : 256; }

// Parts of the reduction of a product with c rows whose smallest tiles (32 x 256) leave CUs idle: half a workgroup per CU, and at
// least two steps of 16 planes each.  own_join: the parts meet in a launch of their own (forward), which pays from a quarter of
// that on (one pixel, c 1024, hidden 4096, bf16: 36 -> 23 us, 64 workgroups: 19.6 -> 21.2; backward at 64 workgroups: 62.5 -> 57.8 us).
static inline unsigned ffn_tile_parts(unsigned pixels, int c, int kp_h, bool own_join) {
    const unsigned workgroups = (pixels + 255) / 256 * ((c + 31) / 32), want = 128 / workgroups, most = (unsigned)kp_h / 32;
    if (want < (own_join ? 4u : 2u) || most < 2) return 1;
    return want < most ? want : most;
}

// Rows of the hidden biases' partial sums that are added at a time (0: all at once): from 512 rows on 256, or as many as leave 1024 sums
static inline unsigned ffn_bias_fold(unsigned rows) { return rows <= 512 ? 0 : rows <= 256 * 1024 ? 256 : (rows + 1023) / 1024; }

constexpr int kFfnFusedPlanes = 16, kFfnBackPlanes = 12;
constexpr unsigned kFfnBackTile = 128, kFfnBackTileWide = 256;  // pixels of its workgroups, up to kFfnBackPlanes planes and beyond

// The launches of one compute type
struct FfnLaunch {
    int (*gemm)(const FfnParams& p, int what, int act, hipStream_t s);
    int (*fused)(const FfnParams& p, unsigned parts, int act, hipStream_t s);  // up to kFfnFusedPlanes planes of channels
    int (*join)(const FfnParams& p, int parts, hipStream_t s);
    int (*back)(const FfnParams& p, unsigned parts, int act, hipStream_t s);  // up to kFfnFusedPlanes planes; with dx up to kFfnBackPlanes
    int (*wgrad)(const FfnParams& p, unsigned splits, hipStream_t s);
    int (*finish)(FfnFinish f, hipStream_t s);
    int (*transpose)(const FfnParams& p, hipStream_t s);
};

}  // namespace srmi

const srmi::FfnLaunch* srmi_ffn_f16();
const srmi::FfnLaunch* srmi_ffn_bf16();
const srmi::FfnLaunch* srmi_ffn_f32();
