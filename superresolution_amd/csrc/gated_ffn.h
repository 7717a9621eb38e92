// What the gated feed-forward block's host code (gated_ffn.hip) and its kernels (gated_ffn_kernel.h, one translation unit per
// compute type) share.
#pragma once
#include "common.h"

namespace srmi {

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
    char *hid, *dg, *du;              // [plane of hidden][pixel of the launch][32 bytes]
    float* part;                      // [hidden part][pixel][c]: partial outputs of the one-launch form (null: it writes out)
    float* bias_part;                 // [pixel tile][2][hidden]
    // weight gradients
    float* wpart;                     // [split][3 * hidden * c]
    unsigned split_pixels;
};

// What a launch of the block's tile kernel computes
enum {
    kFfnHidden = 0,      // hid = act(w_gate x + b_gate) * (w_up x + b_up)
    kFfnDown = 1,        // out = res + res_scale * (w_down hid + b_down)
    kFfnHiddenGrad = 2,  // hid, dg, du from x and dy
    kFfnInputGrad = 3    // out = wt_gate dg + wt_up du
};

constexpr int kFfnFusedPlanes = 16, kFfnBackPlanes = 12;
constexpr unsigned kFfnBackTile = 128, kFfnBackTileWide = 256;  // pixels of its workgroups, up to kFfnBackPlanes planes and beyond

// The launches of one compute type
struct FfnLaunch {
    int (*gemm)(const FfnParams& p, int what, int act, hipStream_t s);
    int (*fused)(const FfnParams& p, unsigned parts, int act, hipStream_t s);  // up to kFfnFusedPlanes planes of channels
    int (*join)(const FfnParams& p, int parts, hipStream_t s);
    int (*back)(const FfnParams& p, int act, hipStream_t s);  // up to kFfnFusedPlanes planes; with dx up to kFfnBackPlanes
    int (*wgrad)(const FfnParams& p, unsigned splits, hipStream_t s);
    int (*wjoin)(const FfnParams& p, int splits, void* g_gate, void* g_up, void* g_down, hipStream_t s);
    int (*dbias)(const FfnParams& p, unsigned run, float* part, hipStream_t s);
    int (*transpose)(const FfnParams& p, hipStream_t s);
};

}  // namespace srmi

const srmi::FfnLaunch* srmi_ffn_f16();
const srmi::FfnLaunch* srmi_ffn_bf16();
const srmi::FfnLaunch* srmi_ffn_f32();
