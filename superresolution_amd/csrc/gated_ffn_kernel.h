// Kernels of the gated feed-forward block (template over the compute type).  Included by one translation unit per type
// (gated_ffn_f16.hip, _bf16, _f32); the host entry points are in gated_ffn.hip.
//
//   hid = act(w_gate x + b_gate) * (w_up x + b_up)        out = res + res_scale * (w_down hid + b_down)
//
// MFMA roles as in the convolutions: A operand = weights (rows = output channels), B operand = pixels (columns).  A plane
// holds 32 bytes of channels per pixel, exactly one 32x32x16 half (or four 32x32x2 f32) B operand for 32 pixels with lane l
// taking bytes 16 * (l / 32) of pixel l % 32: pixel operands go from memory (or from the accumulators of the product before) straight to registers,
// 1 KiB contiguous per wave and plane, and never through LDS.  Weights, which all waves of a workgroup share, go through LDS.
//
// The accumulator of a 32x32 product holds, in lane l and register i, row 8 * (i / 4) + 4 * (l / 32) + i % 4 of column l % 32.
// For the half types the rows of a weight block are therefore fed in the order that swaps bits 2 and 3 of the row number:
// registers 8q .. 8q + 7 then hold channels 16q + 8 * (l / 32) + 0 .. 7, one 16-byte piece of plane q: a store, or
// after rounding the B operand of the next product, without any exchange between lanes.  For f32 (8 channels per plane) the
// natural order already does that with registers 4q .. 4q + 3.
#pragma once
#include <atomic>
#include <type_traits>

#include "common.h"
#include "devutil.h"
#include "gated_ffn.h"

namespace srmi {

template <int DT>
struct FfnType {
    static constexpr int ES = DT == SRMI_F32 ? 4 : 2;
    static constexpr int CPB = 32 / ES;   // channels of a plane
    static constexpr int E = 16 / ES;     // channels of a 16-byte piece
    static constexpr int NQ = 32 / CPB;   // planes of a 32-row block
};

// Hidden tensors in the workspace: blocks of 64 pixels, [block][plane][pixel][32 bytes].  What a step of the weight gradients
// reads is then one contiguous range (plane after plane over all pixels it would be a separate page for every plane).
constexpr int kFfnHiddenPlane = kFfnHiddenBlock * 32;  // bytes between the planes of a block
__device__ __forceinline__ unsigned long long ffn_hidden_pixel(unsigned m, int planes) {
    return (unsigned long long)(m / kFfnHiddenBlock) * ((unsigned long long)planes * kFfnHiddenPlane) + (m % kFfnHiddenBlock) * 32;
}

#if defined(__HIP_DEVICE_COMPILE__)

__device__ __forceinline__ __amdgpu_buffer_rsrc_t ffn_rsrc(const void* base, unsigned bytes) {
    return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (int)bytes, 0x00020000);
}

template <int DT>
__device__ __forceinline__ void ffn_mma(f32x16& c, const u32x4& a, const u32x4& b) {
    if constexpr (DT == SRMI_F16) {
        c = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    } else if constexpr (DT == SRMI_BF16) {
        c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    } else {
        const f32x4 av = __builtin_bit_cast(f32x4, a), bv = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(av[j], bv[j], c, 0, 0, 0);
    }
}

// E accumulator values -> a 16-byte piece, rounded to nearest even (f16 saturating)
template <int DT>
__device__ __forceinline__ u32x4 ffn_pack(const float* v) {
    if constexpr (DT == SRMI_F32) {
        return __builtin_bit_cast(u32x4, f32x4{v[0], v[1], v[2], v[3]});
    } else if constexpr (DT == SRMI_F16) {
        // the cast overflows to infinity, the packed minimum and maximum (which keep NaN) bring it back to +-65504
        f16x8 h;
#pragma unroll
        for (int j = 0; j < 8; ++j) h[j] = (_Float16)v[j];
        const _Float16 top = (_Float16)65504.f;
        const f16x8 hi = {top, top, top, top, top, top, top, top};
        h = __builtin_elementwise_minimum(__builtin_elementwise_maximum(h, -hi), hi);
        return __builtin_bit_cast(u32x4, h);
    } else {
        bf16x8 h;
#pragma unroll
        for (int j = 0; j < 8; ++j) h[j] = (__bf16)v[j];
        return __builtin_bit_cast(u32x4, h);
    }
}

template <int DT>
__device__ __forceinline__ void ffn_unpack(const u32x4& u, float* v) {
    if constexpr (DT == SRMI_F32) {
        const f32x4 h = __builtin_bit_cast(f32x4, u);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = h[j];
    } else if constexpr (DT == SRMI_F16) {
        const f16x8 h = __builtin_bit_cast(f16x8, u);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (float)h[j];
    } else {
        const bf16x8 h = __builtin_bit_cast(bf16x8, u);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (float)h[j];
    }
}

// Row of a 32-row weight block that operand row r takes (see the head of the file)
template <int DT>
__device__ __forceinline__ int ffn_row(int r) {
    return DT == SRMI_F32 ? r : (r & 0x13) | ((r & 4) << 1) | ((r & 8) >> 1);
}

// ---- activations ---------------------------------------------------------------------------------------------------------
// sigmoid through the hardware's exp2 and reciprocal (1 ulp each): exp2 overflows to inf for very negative a, and 1 / inf = 0
__device__ __forceinline__ float ffn_sigmoid(float a) {
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(a * -1.44269504088896341f));
}
// GELU, a Phi(a), and its slope from Q(x) = Phi(-x), x = |a|:
//   gelu(a) = max(a, 0) - x Q(x)     gelu'(a) = a < 0 ? D : 1 - D,  D = Q(x) - x exp(-x^2 / 2) / sqrt(2 pi)
// so that the error scales with the value on both sides of zero and in the tail.  (As 1/2 plus something, or with t = 1 / (1 + k x) and x t as
// (1 - t) / k, an absolute error of an ulp of 1 is left: with gates around 1e-3 that is 1.6e-4 of the result.)  The polynomials are minimax
// fits of the relative error of Q, made here in 64 bits.
// Half types: Q(x) = exp2(polynomial of degree 9), whose error of 1e-6 at 0, 1e-5 at 4 and 4.5e-4 from 6 to 11 is what these types
// cannot hold (half steps 5e-4 and 4e-3; f16's smallest value, 6e-8, is gelu(-5.6)); beyond 11, where x Q(x) = 2e-27, x counts as 11.  One
// exponential and no reciprocal (quarter rate each): 339 x 510 x 64, hidden 128, f16: 24.0 us, 25.3 with P and t as below.
// f32: Q(x) = t P(t) exp(-x^2 / 2), t = 1 / (1 + k x), P of degree 7, 8e-9 for x >= 1; below, where the rounding of 1 + k x alone would cost 4
// ulp, Q(x) = 1/2 - x R(x^2), 7e-10.  The exponent's rounding, |x^2 / 2| 2^-24 of the result, is added back.  On normal arguments the rms
// error is 2.9e-8, with erf in f32 3.8e-8.  Beyond x = 32 Q and the exponential are 0, so x counts as 32.
__device__ __forceinline__ float ffn_poly(float t, float c) { return c; }
template <typename... C>
__device__ __forceinline__ float ffn_poly(float t, float c, C... more) { return __builtin_fmaf(ffn_poly(t, more...), t, c); }
constexpr float kHalfLog2e = 0.72134752044448170f;
// x, Q(x) and (SLOPE) exp(-x^2 / 2)
template <int DT, bool SLOPE>
__device__ __forceinline__ void ffn_gelu_tail(float a, float& x, float& q, float& ex) {
    x = __builtin_elementwise_minimum(fabsf(a), DT == SRMI_F32 ? 32.f : 11.f);  // NaN stays NaN
    if constexpr (DT == SRMI_F32) {
        const float s = x * x, p = s * -kHalfLog2e, e = __builtin_amdgcn_exp2f(p);
        // what -x^2 log2(e) / 2 has beyond p: log2(e) / 2 = kHalfLog2e + 9.629815e-9
        const float r = __builtin_fmaf(s, -9.629815e-9f, __builtin_fmaf(__builtin_fmaf(x, x, -s), -kHalfLog2e, __builtin_fmaf(s, -kHalfLog2e, -p)));
        ex = __builtin_fmaf(e, r * 0.69314718055994531f, e);
        const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(x, 0.245f, 1.f));
        const float far = (t * ex) * ffn_poly(t, 0.09775952107f, 0.09734529477f, 0.09545782383f, 0.0620305858f, 0.1192563821f, -0.06129458231f, 0.1429736815f, -0.05354772629f);
        const float near = __builtin_fmaf(-x, ffn_poly(s, 0.3989422801f, -0.06649035992f, 0.009973323411f, -0.001186329944f, 0.0001134863735f, -7.654208682e-06f), 0.5f);
        q = x < 1.f ? near : far;
    } else {
        q = __builtin_amdgcn_exp2f(ffn_poly(x, -0.999998808f, -1.15117445f, -0.458709605f, -0.0536790776f, 0.00835557953f, -0.000886133239f, 5.39448485e-05f, -9.48812329e-07f,
                                            -7.3869869e-08f, 3.25312062e-09f));
        if constexpr (SLOPE) ex = __builtin_amdgcn_exp2f((x * -kHalfLog2e) * x);
    }
}
// (max(a, 0) as the integer maximum of its bits: one instruction, where a float maximum quiets its operand first; NaN comes through x)
__device__ __forceinline__ float ffn_gelu_value(float a, float x, float q) { return __builtin_fmaf(-x, q, __int_as_float(max(__float_as_int(a), 0))); }

template <int DT, int ACT>
__device__ __forceinline__ float ffn_act(float a) {
    if constexpr (ACT == SRMI_ACT_SILU) return a * ffn_sigmoid(a);
    else if constexpr (ACT == SRMI_ACT_GELU) {
        float x, q, ex;
        ffn_gelu_tail<DT, false>(a, x, q, ex);
        return ffn_gelu_value(a, x, q);
    } else if constexpr (ACT == SRMI_ACT_RELU) return a < 0.f ? 0.f : a;
    else if constexpr (ACT == SRMI_ACT_LRELU) return a < 0.f ? 0.2f * a : a;
    else return a;
}
template <int DT, int ACT>
__device__ __forceinline__ float ffn_act_slope(float a, float& slope) {
    if constexpr (ACT == SRMI_ACT_SILU) {
        const float s = ffn_sigmoid(a);
        slope = s * (1.f + a * (1.f - s));
        return a * s;
    } else if constexpr (ACT == SRMI_ACT_GELU) {
        float x, q, ex;
        ffn_gelu_tail<DT, true>(a, x, q, ex);
        const float d = __builtin_fmaf(x * -0.39894228040143268f, ex, q);
        slope = a < 0.f ? d : 1.f - d;
        return ffn_gelu_value(a, x, q);
    } else if constexpr (ACT == SRMI_ACT_RELU) {
        slope = a > 0.f ? 1.f : 0.f;
        return a < 0.f ? 0.f : a;
    } else if constexpr (ACT == SRMI_ACT_LRELU) {
        slope = a > 0.f ? 1.f : 0.2f;
        return a < 0.f ? 0.2f * a : a;
    } else {
        slope = 1.f;
        return a;
    }
}

// ---- weight tile: ROWS rows x 128 bytes of the reduction, global -> LDS by LDS-DMA ---------------------------------------
// The 16-byte piece s of row r sits in slot 8 * r + (s ^ key(r)), key(r) = bits 1, 2, 3 of r in reverse order: the 16-lane
// groups of a ds_read_b128 (16 rows, one piece) touch 16 different bank groups, and so do the half waves of a transposed
// read (4 rows, four pieces).  Rows and bytes beyond the matrix read as zeros.
__device__ __forceinline__ int ffn_key(int r) { return ((r & 2) << 1) | ((r & 4) >> 1) | ((r & 8) >> 3); }
// A lane's offset in a tile (of a row of 8 per piece) is fixed for a wave, the rest of the address is uniform.  ld: bytes of a row.
constexpr unsigned kFfnBeyond = 0x80000000u;  // past every matrix (at most 2^28 bytes), also with a uniform offset added
__device__ __forceinline__ unsigned ffn_lane_offset(unsigned ld, int wave, int lane) {  // wave: its parity is that of its pieces
    return (unsigned)(lane >> 3) * ld + (unsigned)((lane & 7) ^ ffn_key((lane >> 3) | ((wave & 1) << 3))) * 16u;
}
__device__ __forceinline__ unsigned ffn_lane_byte(int wave, int lane) { return (unsigned)((lane & 7) ^ ffn_key((lane >> 3) | ((wave & 1) << 3))) * 16u; }
template <int NW, int ROWS>
__device__ __forceinline__ void ffn_stage(const __amdgpu_buffer_rsrc_t rsrc, unsigned offset, unsigned row0, unsigned byte0, unsigned ld, char* lds, int wave) {
    static_assert(NW % 2 == 0, "");
#pragma unroll
    for (int i = 0; i < (ROWS / 8 + NW - 1) / NW; ++i) {
        const int k = wave + NW * i;
        if (ROWS / 8 % NW != 0 && k >= ROWS / 8) break;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)(lds + k * 1024), 16, offset + ((row0 + 8 * k) * ld + byte0), 0, 0, 0);
    }
}
// The A operand of 32 rows and plane k of the tile (128 bytes, so four planes, per row): `at` = this lane's place in the first
// 32 rows of the tile (ffn_lane_rows), whose piece number the plane's enters as an exclusive or; `more`: further rows and tiles.
template <int DT>
__device__ __forceinline__ unsigned ffn_lane_rows(int lane) {
    const int r = ffn_row<DT>(lane & 31);
    return (unsigned)(8 * r + ((lane >> 5) ^ ffn_key(r))) * 16u;
}
__device__ __forceinline__ u32x4 ffn_weights(const char* smem, unsigned at, int k, unsigned more) { return *(const u32x4*)(smem + ((at ^ (unsigned)(32 * k)) + more)); }
// Keeps a value from being computed ahead of a loop and held in a register through it
__device__ __forceinline__ unsigned ffn_here(unsigned v) {
    asm volatile("" : "+v"(v));
    return v;
}

// Every LDS-DMA and LDS read of this wave has landed, then all waves meet.
__device__ __forceinline__ void ffn_meet() {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
}

// The same, but the wave's YOUNGER latest vector-memory operations (stores issued after the LDS-DMA it waits for) may still run:
// operations complete in the order they were issued.
template <int YOUNGER>
__device__ __forceinline__ void ffn_meet_but() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(YOUNGER) : "memory");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
}

// Sums of 16 registers over the 32 lanes of each half wave, spread: lane l returns the sum of register r(l) of its half, r =
// bits 4, 3, 2, 1 of l read as bits 3, 2, 1, 0.  Each step adds what half of the lanes hold of one register to the other
// half's and keeps one register where there were two: 16 + 3 * (4 + 2 + 1) + 2 operations instead of 16 sums of 5.
template <int CTRL>
__device__ __forceinline__ float ffn_dpp_all(float v) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false)); }
__device__ __forceinline__ float ffn_spread_sums(const float (&v)[16], int lane) {
    float a[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        // rows 0, 2 keep register i, rows 1, 3 register i + 8
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[i]), __float_as_uint(v[i + 8]), false, false);
        a[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    float b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float s = a[i] + ffn_dpp_all<0x128>(a[i]), t = a[i + 4] + ffn_dpp_all<0x128>(a[i + 4]);  // row_ror:8
        b[i] = lane & 8 ? t : s;
    }
    float c[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float s = b[i] + ffn_dpp_all<0x141>(b[i]), t = b[i + 2] + ffn_dpp_all<0x141>(b[i + 2]);  // row_half_mirror: lane ^ 7
        c[i] = lane & 4 ? t : s;
    }
    // lanes l and l ^ 7 have met: what is left lies in bits 0, 1 against the mirrored lane's, so two more steps over a quad
    const float s = c[0] + ffn_dpp_all<0x4e>(c[0]), t = c[1] + ffn_dpp_all<0x4e>(c[1]);  // quad_perm [2,3,0,1]
    const float d = lane & 2 ? t : s;
    return d + ffn_dpp_all<0xb1>(d);  // quad_perm [1,0,3,2]
}
#endif

#if defined(__HIP_DEVICE_COMPILE__)
// A piece of a part's sums: [part][plane][pixel][channel of the plane] in f32, so that a wave's lanes write (and the join reads)
// consecutive addresses
template <int DT>
__device__ __forceinline__ void ffn_store_part(const FfnParams& p, unsigned part, int plane, unsigned m, int lh, const f32x16& v, int at) {
    using T = FfnType<DT>;
    float* d = p.part + (((unsigned long long)part * p.kp_c + plane) * (p.m - p.m0) + (m - p.m0)) * T::CPB + lh * T::E;
#pragma unroll
    for (int e = 0; e < T::E; e += 4) *(f32x4*)(d + e) = f32x4{v[at + e], v[at + e + 1], v[at + e + 2], v[at + e + 3]};
}
#endif

template <int WHAT, int RB_>
struct FfnShape {
    static constexpr int NA = WHAT == kFfnHidden ? 2 : WHAT == kFfnHiddenGrad ? 3 : 1;  // products at once
    static constexpr int RB = RB_;                                                      // 32-row blocks of each
    static constexpr int NS = WHAT == kFfnHiddenGrad ? 2 : 1;                           // pixel operands at once
    static constexpr int NW = 8;                                                        // waves
    static constexpr int ROWS = RB * 32;
    static constexpr int PIXELS = NW * 32;                                              // of a workgroup
    static constexpr int TP = RB > 1 ? 1 : NS == 2 ? 2 : 4;                             // column tiles (four planes) of a step
    static constexpr int TILE = NA * ROWS * 128;
    static constexpr int STAGE = TP * TILE;
};

// One tile of ROWS rows x 256 pixels (8 waves of 32) of NA products that share their rows' index and reduction.  The reduction runs in steps
// of TP times four planes (128 bytes of a weight row): weights double-buffered in LDS, pixels in registers, both requested one step
// ahead, one barrier per step.  Measured: dx of 131072 pixels, c 256, hidden 1024, bf16: 185 to 195 us = 705 to 743 TFLOP/s with 0.55 GB of dg and du read.
// A step of a tile of 32 rows has so little to multiply that it would wait for its successor's loads;
// there is room in LDS and registers for longer ones.  blockIdx.z splits the reduction of the products with c rows where such tiles
// are few; the parts leave f32 partial sums that are added in order behind it.
template <int DT, int WHAT, int RB_, int ACT>
__global__ __launch_bounds__(512, 2) void ffn_gemm_kernel(const FfnParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
    using T = FfnType<DT>;
    using S = FfnShape<WHAT, RB_>;
    constexpr int NA = S::NA, RB = S::RB, NS = S::NS, NW = S::NW, TP = S::TP;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lh = lane >> 5;
    const unsigned row0 = blockIdx.y * S::ROWS;
    const bool to_hidden = WHAT == kFfnHidden || WHAT == kFfnHiddenGrad;
    const unsigned rows = to_hidden ? p.hidden : p.c;
    const int kp = to_hidden ? p.kp_c : p.kp_h;
    const unsigned ld = (unsigned)kp * 32u;

    // this lane's pixel; one beyond the launch's last reads the last one and is not stored
    unsigned m = p.m0 + blockIdx.x * S::PIXELS + wave * 32 + (lane & 31);
    const bool mine = m < p.m;
    if (!mine) m = p.m - 1;
    const unsigned img = (__umulhi(m, p.hw_mul) + m) >> p.hw_shift, pix = m - img * p.hw;
    const bool busy = p.m0 + blockIdx.x * S::PIXELS + wave * 32 < p.m;  // a wave without pixels only helps to stage the weights
    auto pixel_at = [&](const TView& t) { return t.ptr + (long long)img * t.img_stride_b + (unsigned long long)pix * 32 + lh * 16; };
    auto hidden_at = [&](char* base) { return base + ffn_hidden_pixel(m - p.m0, p.kp_h) + lh * 16; };

    const char* src[NS];
    const int steps_each = (kp + 4 * TP - 1) / (4 * TP);
    const int steps_all = WHAT == kFfnInputGrad ? 2 * steps_each : steps_each;
    // blockIdx.z: a part of the reduction
    const int begin = (int)((unsigned)steps_all * blockIdx.z / gridDim.z), steps = (int)((unsigned)steps_all * (blockIdx.z + 1) / gridDim.z);
    auto set_source = [&](int pair) {
        if constexpr (WHAT == kFfnHidden) src[0] = pixel_at(p.x);
        if constexpr (WHAT == kFfnDown) src[0] = hidden_at(p.hid);
        if constexpr (WHAT == kFfnHiddenGrad) { src[0] = pixel_at(p.x); src[NS - 1] = pixel_at(p.dy); }
        if constexpr (WHAT == kFfnInputGrad) src[0] = hidden_at(pair ? p.du : p.dg);
    };
    auto plane_of = [&](int i) { return to_hidden ? (i ? p.dy.plane_stride_b : p.x.plane_stride_b) : (long long)kFfnHiddenPlane; };

    const unsigned lane_rows = ffn_lane_rows<DT>(lane);
    const unsigned lane_offset = ffn_lane_offset(ld, wave, lane), lane_byte = ffn_lane_byte(wave, lane);
    auto stage = [&](int step, int buf) {
        const int pair = WHAT == kFfnInputGrad && step >= steps_each ? 1 : 0;
        char* lds = smem + buf * S::STAGE;
        auto one = [&](const char* w, int at) {
#pragma unroll
            for (int t = 0; t < TP; ++t) {
                const unsigned byte0 = (unsigned)((step - pair * steps_each) * TP + t) * 128u;
                ffn_stage<NW, S::ROWS>(ffn_rsrc(w, rows * ld), byte0 + lane_byte < ld ? lane_offset : kFfnBeyond, row0, byte0, ld, lds + t * S::TILE + at * S::ROWS * 128, wave);
            }
        };
        if constexpr (WHAT == kFfnHidden || WHAT == kFfnHiddenGrad) {
            one(p.w_gate, 0);
            one(p.w_up, 1);
            if constexpr (WHAT == kFfnHiddenGrad) one(p.wt_down, 2);
        } else {
            one(WHAT == kFfnDown ? p.w_down : pair ? p.wt_up : p.wt_gate, 0);
        }
    };
    auto fetch = [&](int step, u32x4 (&b)[NS][4 * TP]) {
        const int pair = WHAT == kFfnInputGrad && step >= steps_each ? 1 : 0;
        if (WHAT == kFfnInputGrad && step == steps_each) set_source(1);
        const int plane0 = (step - pair * steps_each) * 4 * TP;
#pragma unroll
        for (int i = 0; i < NS; ++i)
#pragma unroll
            for (int k = 0; k < 4 * TP; ++k) {
                if (plane0 + k < kp) b[i][k] = *(const u32x4*)(src[i] + (plane0 + k) * plane_of(i));
                else b[i][k] = u32x4{0u, 0u, 0u, 0u};
            }
    };

    f32x16 acc[NA][RB];
#pragma unroll
    for (int a = 0; a < NA; ++a)
#pragma unroll
        for (int r = 0; r < RB; ++r)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[a][r][i] = 0.f;

    u32x4 cur[NS][4 * TP], nxt[NS][4 * TP];
    set_source(begin >= steps_each);
    stage(begin, begin & 1);
    fetch(begin, cur);
    for (int step = begin; step < steps; ++step) {
        ffn_meet();
        if (step + 1 < steps) {
            stage(step + 1, (step + 1) & 1);
            fetch(step + 1, nxt);
        }
        if (busy) {
            // operands read three ahead of their multiplies
            constexpr int N = 4 * TP * NA * RB, AHEAD = 3;
            const unsigned at = ffn_here(lane_rows + (step & 1) * S::STAGE);
            u32x4 w[AHEAD + 1];
            auto read = [&](int i) { w[i % (AHEAD + 1)] = ffn_weights(smem, at, i / (NA * RB) % 4, i / (4 * NA * RB) * S::TILE + (i % (NA * RB)) * 4096); };
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) read(i);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if (i + AHEAD < N) read(i + AHEAD);
                __builtin_amdgcn_sched_barrier(0);
                const int a = i / RB % NA;
                ffn_mma<DT>(acc[a][i % RB], w[i % (AHEAD + 1)], cur[WHAT == kFfnHiddenGrad && a == 2 ? NS - 1 : 0][i / (NA * RB)]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
#pragma unroll
        for (int i = 0; i < NS; ++i)
#pragma unroll
            for (int k = 0; k < 4 * TP; ++k) cur[i][k] = nxt[i][k];
    }

    // ---- epilogue: E channels ch .. ch + E - 1 of the pixel per 16-byte piece --------------------------------------------------
    constexpr int E = T::E;
    if constexpr (WHAT == kFfnHiddenGrad) {
        if (p.bias_part) ffn_meet();  // the stage buffers are free for the sums
    }
#pragma unroll
    for (int r = 0; r < RB; ++r) {
        float gsum[16], usum[16];
        if constexpr (WHAT == kFfnHiddenGrad) {
#pragma unroll
            for (int i = 0; i < 16; ++i) gsum[i] = usum[i] = 0.f;
        }
#pragma unroll
        for (int k = 0; k < T::NQ; ++k) {
            const unsigned plane = (row0 + r * 32) / T::CPB + k;
            const unsigned ch = plane * T::CPB + lh * E;
            if (plane * T::CPB >= rows) continue;
            float bg[E], bu[E];
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if constexpr (WHAT == kFfnHidden || WHAT == kFfnHiddenGrad) {
                    bg[e] = p.b_gate ? p.b_gate[ch + e] : 0.f;
                    bu[e] = p.b_up ? p.b_up[ch + e] : 0.f;
                }
                if constexpr (WHAT == kFfnDown) bg[e] = p.b_down && blockIdx.z == 0 ? p.b_down[ch + e] : 0.f;
            }
            float v[E], g[E], u[E];
            if constexpr (WHAT == kFfnHidden) {
#pragma unroll
                for (int e = 0; e < E; ++e) v[e] = ffn_act<DT, ACT>(acc[0][r][k * E + e] + bg[e]) * (acc[1][r][k * E + e] + bu[e]);
                if (mine) *(u32x4*)(hidden_at(p.hid) + plane * kFfnHiddenPlane) = ffn_pack<DT>(v);
            } else if constexpr (WHAT == kFfnHiddenGrad) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    float slope;
                    const float up = acc[1][r][k * E + e] + bu[e];
                    const float a = ffn_act_slope<DT, ACT>(acc[0][r][k * E + e] + bg[e], slope);
                    const float dh = p.res_scale * acc[NA - 1][r][k * E + e];
                    v[e] = a * up;
                    g[e] = dh * up * slope;
                    u[e] = dh * a;
                    gsum[k * E + e] = mine ? g[e] : 0.f;
                    usum[k * E + e] = mine ? u[e] : 0.f;
                }
                if (mine) {
                    *(u32x4*)(hidden_at(p.hid) + plane * kFfnHiddenPlane) = ffn_pack<DT>(v);
                    *(u32x4*)(hidden_at(p.dg) + plane * kFfnHiddenPlane) = ffn_pack<DT>(g);
                    *(u32x4*)(hidden_at(p.du) + plane * kFfnHiddenPlane) = ffn_pack<DT>(u);
                }
            } else {
                if (RB == 1 && p.part) {
                    if constexpr (WHAT == kFfnDown) {
#pragma unroll
                        for (int e = 0; e < E; ++e) acc[0][r][k * E + e] += bg[e];
                    }
                    if (mine) ffn_store_part<DT>(p, blockIdx.z, plane, m, lh, acc[0][r], k * E);
                    continue;
                }
                if constexpr (WHAT == kFfnDown) {
#pragma unroll
                    for (int e = 0; e < E; ++e) v[e] = p.res_scale * (acc[0][r][k * E + e] + bg[e]);
                    if (p.res.ptr) {
                        ffn_unpack<DT>(*(const u32x4*)(pixel_at(p.res) + plane * p.res.plane_stride_b), u);
#pragma unroll
                        for (int e = 0; e < E; ++e) v[e] += u[e];
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < E; ++e) v[e] = acc[0][r][k * E + e];
                }
                if (mine) *(u32x4*)(pixel_at(p.out) + plane * p.out.plane_stride_b) = ffn_pack<DT>(v);
            }
        }
        if constexpr (WHAT == kFfnHiddenGrad) {
            if (p.bias_part) {
                const float a = ffn_spread_sums(gsum, lane), b = ffn_spread_sums(usum, lane);
                const int i = (lane >> 1) & 15, ch = r * 32 + T::CPB * (i / E) + E * lh + i % E;
                float* red = (float*)smem + wave * 2 * S::ROWS;
                if (!(lane & 1)) { red[ch] = a; red[S::ROWS + ch] = b; }
            }
        }
    }
    if constexpr (WHAT == kFfnHiddenGrad) {
        if (p.bias_part) {
            __syncthreads();
            const float* red = (const float*)smem;
            for (int i = threadIdx.x; i < 2 * S::ROWS; i += 64 * NW) {
                const unsigned ch = row0 + i % S::ROWS;
                if (ch >= rows) continue;
                float v = red[i];
#pragma unroll
                for (int w = 1; w < NW; ++w) v += red[w * 2 * S::ROWS + i];
                p.bias_part[((unsigned long long)blockIdx.x * 2 + i / S::ROWS) * rows + ch] = v;
            }
        }
    }
#endif
}

// ---- the whole block in one launch ---------------------------------------------------------------------------------------
// A wave keeps its pixels' inputs (KP planes) and all output channels in registers and walks the hidden units in chunks of
// 32: both products of a chunk, activation and product in the accumulators, which as 16-byte pieces are the B operand of the
// second product.  Hidden values never leave the registers; the only traffic is x, res and out once, and the weights of a
// chunk (double-buffered in LDS by LDS-DMA), which stay in L2.
// With few pixels blockIdx.y splits the hidden units; the parts leave f32 partial sums that ffn_join_kernel adds in order.
// Why one pass: 8 x 256 x 256 pixels, c 256, hidden 512 would move 1 GB of hidden values and back; so x, res and out (0.8 GB) are all.
// Measured, from card to card: that size in bf16 450 to 494 us = 918 to 834 TFLOP/s, at the card's power limit (a library product of 8192^3:
// 1107 to 1150); f32, 65536 pixels, c 64, hidden 256: 56 to 63 us = 115 to 103 TFLOP/s (147 to 136); f16, 339 x 510, c 64, hidden 128, gelu: 22
// to 25 us against 14 us for a copy of its bytes (two rounds of workgroups whose first loads nothing hides); one pixel, c 256, hidden 512: 10 us in two launches.
// Eight waves of 32 pixels beyond 12 planes: with four of 64 pixels, which read the weights from LDS half as often, 738 instead
// of 569 us at the first size (one wave per SIMD, and nothing runs under the activations).
template <int DT, int KP, int NW>
struct FfnFused {
    using T = FfnType<DT>;
    static constexpr int KT = (KP + 3) / 4;                     // 128-byte column tiles of w_gate / w_up
    static constexpr int RB = (KP + T::NQ - 1) / T::NQ;         // 32-row blocks of w_down
    static constexpr int UP = KT * 32 * 128;                    // bytes of a chunk of w_gate or w_up
    static constexpr int DOWN = RB * 32 * 32 * T::ES;           // bytes of a chunk of w_down
    static constexpr int STAGE = 2 * UP + DOWN;                  // then the chunk's biases of gate and up, 256 bytes each
    static constexpr int SLOT = STAGE + 512;
    static constexpr int PIXELS = NW * 32;
    // Registers, about, and the waves per SIMD they leave; eight waves of a workgroup are two per SIMD whatever they need.  At KP = 16 the half
    // types need more than the 256 of that: 12 registers (19 with GELU) that the chunk loop does not use wait in scratch while it runs, and
    // with GELU one is read back per chunk.
    static constexpr int REGS = KP * 4 + RB * 16 + 32 + 64;
    static constexpr int WAVES = REGS <= 128 ? 4 : REGS <= 168 ? 3 : REGS <= 256 || NW == 8 ? 2 : 1;
};

#if defined(__HIP_DEVICE_COMPILE__)
// A chunk's three weight tiles, and behind them its biases (zeros where there are none, then 32 more that nobody reads).
// The tile of w_down is ROWS rows x 32 hidden units.  Half types: 64 bytes per row, piece s of row r in slot 4 r + (s ^ ((r >> 2) &
// 3)), again 16 bank groups for 16 rows; f32 rows are 128 bytes and lie as those of the other two.
template <int DT, int KP, int NW>
struct FfnStager {
    using S = FfnFused<DT, KP, NW>;
    unsigned ld_up, ld_down, up, up_last, down, down_byte;
    __device__ __forceinline__ FfnStager(const FfnParams& p, int wave, int lane) {
        ld_up = (unsigned)p.kp_c * 32u;
        ld_down = (unsigned)p.kp_h * 32u;
        up = ffn_lane_offset(ld_up, wave, lane);
        up_last = (S::KT - 1) * 128u + ffn_lane_byte(wave, lane) < ld_up ? up : kFfnBeyond;
        if constexpr (DT == SRMI_F32) {
            down = ffn_lane_offset(ld_down, wave, lane);
            down_byte = ffn_lane_byte(wave, lane);
        } else {
            down_byte = (unsigned)((lane & 3) ^ ((lane >> 4) & 3)) * 16u;
            down = (unsigned)(lane >> 2) * ld_down + down_byte;
        }
    }
    __device__ __forceinline__ void run(const FfnParams& p, int chunk, char* lds, int wave, int lane) const {
        const auto gate = ffn_rsrc(p.w_gate, p.hidden * ld_up), upper = ffn_rsrc(p.w_up, p.hidden * ld_up), lower = ffn_rsrc(p.w_down, p.c * ld_down);
#pragma unroll
        for (int t = 0; t < S::KT; ++t) {
            const unsigned o = t == S::KT - 1 ? up_last : up;
            ffn_stage<NW, 32>(gate, o, chunk * 32u, t * 128, ld_up, lds + t * 4096, wave);
            ffn_stage<NW, 32>(upper, o, chunk * 32u, t * 128, ld_up, lds + S::UP + t * 4096, wave);
        }
        const unsigned byte0 = (unsigned)chunk * (32u * FfnType<DT>::ES), o = byte0 + down_byte < ld_down ? down : kFfnBeyond;
        char* at = lds + 2 * S::UP;
        if constexpr (DT == SRMI_F32) {
            ffn_stage<NW, S::RB * 32>(lower, o, 0, byte0, ld_down, at, wave);
        } else {
#pragma unroll
            for (int i = 0; i < (S::RB * 2 + NW - 1) / NW; ++i) {
                const int k = wave + NW * i;
                if (S::RB * 2 % NW != 0 && k >= S::RB * 2) break;
                __builtin_amdgcn_raw_ptr_buffer_load_lds(lower, (__attribute__((address_space(3))) void*)(at + k * 1024), 16, o + (16 * k * ld_down + byte0), 0, 0, 0);
            }
        }
        if (wave < 2) {
            const float* b = wave ? p.b_up : p.b_gate;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(ffn_rsrc(b, b ? p.hidden * 4u : 0u), (__attribute__((address_space(3))) void*)(lds + S::STAGE + wave * 256), 4,
                                                     (chunk * 32 + lane) * 4, 0, 0, 0);
        }
    }
};
// This lane's place in the first 32 rows of a tile of w_down; further blocks of 32 rows are kRows bytes on
template <int DT>
struct FfnDownTile {
    static constexpr unsigned kRows = 32 * 32 * FfnType<DT>::ES;
    static __device__ __forceinline__ unsigned lane(int lane) {
        if constexpr (DT == SRMI_F32) return ffn_lane_rows<DT>(lane);
        const int r = ffn_row<DT>(lane & 31);
        return (unsigned)(4 * r + ((lane >> 5) ^ ((r >> 2) & 3))) * 16u;
    }
};

// The two products of a chunk: g += w_gate x, u += w_up x.  Operands are read AHEAD steps before their multiplies (as many as the
// registers allow); left to itself the compiler reads each one right before its use, and the matrix pipe waits out the LDS latency every time.
template <int DT, int KP>
__device__ __forceinline__ void ffn_products(f32x16& g, f32x16& u, const u32x4 (&x)[KP], const char* smem, unsigned at, unsigned up) {
    constexpr int AHEAD = KP > 12 ? 1 : 2;
    u32x4 w[AHEAD + 1][2];
    auto read = [&](int k) {
        w[k % (AHEAD + 1)][0] = ffn_weights(smem, at, k % 4, (k / 4) * 4096);
        w[k % (AHEAD + 1)][1] = ffn_weights(smem, at, k % 4, up + (k / 4) * 4096);
    };
#pragma unroll
    for (int k = 0; k < AHEAD && k < KP; ++k) read(k);
#pragma unroll
    for (int k = 0; k < KP; ++k) {
        if (k + AHEAD < KP) read(k + AHEAD);
        __builtin_amdgcn_sched_barrier(0);
        ffn_mma<DT>(g, w[k % (AHEAD + 1)][0], x[k]);
        ffn_mma<DT>(u, w[k % (AHEAD + 1)][1], x[k]);
        __builtin_amdgcn_sched_barrier(0);
    }
}

// y += w_down h, operands read AHEAD before their multiplies, the first ones before the activation (start)
template <int DT, int RB>
struct FfnDown {
    static constexpr int N = RB * FfnType<DT>::NQ, MOST = RB > 6 ? 2 : 3, AHEAD = N < MOST ? N : MOST;
    u32x4 w[AHEAD + 1];
    __device__ __forceinline__ void read(int i, const char* smem, unsigned at) { w[i % (AHEAD + 1)] = ffn_weights(smem, at, i / RB, (i % RB) * FfnDownTile<DT>::kRows); }
    __device__ __forceinline__ void start(const char* smem, unsigned at) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) read(i, smem, at);
        __builtin_amdgcn_sched_barrier(0);
    }
    __device__ __forceinline__ void run(f32x16 (&y)[RB], const u32x4 (&h)[FfnType<DT>::NQ], const char* smem, unsigned at) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (i + AHEAD < N) read(i + AHEAD, smem, at);
            __builtin_amdgcn_sched_barrier(0);
            ffn_mma<DT>(y[i % RB], w[i % (AHEAD + 1)], h[i / RB]);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
};

// A pixel's KP planes, zeros beyond the tensor's and for a lane that has no pixel
template <int KP>
__device__ __forceinline__ void ffn_load_planes(u32x4 (&v)[KP], const char* a, long long plane_stride, int planes, bool mine = true) {
#pragma unroll
    for (int k = 0; k < KP; ++k) {
        v[k] = *(const u32x4*)(a + (k < planes ? k : planes - 1) * plane_stride);
        const unsigned keep = k < planes && mine ? 0xffffffffu : 0u;
        v[k] = v[k] & u32x4{keep, keep, keep, keep};
    }
}

// out = res + scale * y, all residual planes requested before the first is used
template <int DT, int KP, int RB>
__device__ __forceinline__ void ffn_finish_pixel(const FfnParams& p, const f32x16 (&y)[RB], const char* res, char* out, float scale, bool mine) {
    using T = FfnType<DT>;
    u32x4 o[KP];
    if (res) ffn_load_planes<KP>(o, res, p.res.plane_stride_b, p.kp_c);
#pragma unroll
    for (int k = 0; k < KP; ++k) {
        if (k >= p.kp_c) continue;
        float v[T::E], r[T::E];
        if (res) ffn_unpack<DT>(o[k], r);
#pragma unroll
        for (int e = 0; e < T::E; ++e) {
            v[e] = scale * y[k / T::NQ][(k % T::NQ) * T::E + e];
            if (res) v[e] += r[e];
        }
        if (mine) *(u32x4*)(out + k * p.out.plane_stride_b) = ffn_pack<DT>(v);
    }
}

// The accumulators of a chunk's two products start from its biases (32 floats each in LDS).
template <int DT>
__device__ __forceinline__ void ffn_start(f32x16& g, f32x16& u, const char* b_gate, const char* b_up, int lh) {
    using T = FfnType<DT>;
#pragma unroll
    for (int n = 0; n < T::NQ; ++n)
#pragma unroll
        for (int e = 0; e < T::E; e += 4) {
            const int at = (n * T::CPB + lh * T::E + e) * 4;
            const f32x4 a = *(const f32x4*)(b_gate + at), b = *(const f32x4*)(b_up + at);
#pragma unroll
            for (int j = 0; j < 4; ++j) { g[n * T::E + e + j] = a[j]; u[n * T::E + e + j] = b[j]; }
        }
}
#endif

#if defined(__HIP_DEVICE_COMPILE__)
// y = b_down from LDS (RB * 32 floats, zeros where there are none)
template <int DT, int RB>
__device__ __forceinline__ void ffn_start_down(f32x16 (&y)[RB], const char* b_down, int lh) {
    using T = FfnType<DT>;
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
        for (int n = 0; n < T::NQ; ++n)
#pragma unroll
            for (int e = 0; e < T::E; e += 4) {
                const f32x4 b = *(const f32x4*)(b_down + (r * 32 + n * T::CPB + lh * T::E + e) * 4);
#pragma unroll
                for (int j = 0; j < 4; ++j) y[r][n * T::E + e + j] = b[j];
            }
}
#endif

#if defined(__HIP_DEVICE_COMPILE__)
// The planes of a chunk from `left` on (uniform), which lie beyond the last hidden unit, become zeros: an input's infinity makes 0 * infinity
// = NaN of them, and NaN times the zeros of the next product's weights would reach every channel.  A branch that the last
// chunk alone takes; as selects in every chunk it costs 4 % at 339 x 510 x 64, hidden 128.
template <int NQ>
__device__ __forceinline__ void ffn_zero_beyond(u32x4 (&h)[NQ], int left) {
    if (left < NQ) {
        asm volatile("");  // keeps it a branch
#pragma unroll
        for (int n = 1; n < NQ; ++n)
            if (n >= left) h[n] = u32x4{0u, 0u, 0u, 0u};
    }
}
#endif

#if defined(__HIP_DEVICE_COMPILE__)
// What the rounding of E hidden values to h left, rounded itself: with it the second product has them to twice the type's precision.  Nothing where h is
// at the end of the type's range, infinite or NaN.
template <int DT>
__device__ __forceinline__ u32x4 ffn_pack_rest(const float* v, const u32x4& h) {
    constexpr int E = FfnType<DT>::E;
    float r[E];
    ffn_unpack<DT>(h, r);
#pragma unroll
    for (int e = 0; e < E; ++e) r[e] = fabsf(r[e]) < (DT == SRMI_F16 ? 65504.f : __builtin_inff()) ? v[e] - r[e] : 0.f;
    return ffn_pack<DT>(r);
}
#endif

// TWICE: the hidden values of a half type go into the second product as two halves.  A launch of one workgroup's pixels does so, whose hidden units are
// spread over the CUs a chunk or a few each: without a residual their rounding takes outputs 1.4 times as far from exact ones as the output's
// own does, for a single pixel's 256 channels 1.1 to 1.7 times.  One pixel, c 256, hidden 512, f16: 16 to 17 us either way; at eight workgroups'
// pixels it cost 6 % (1000 pixels, c 192, hidden 1504: 18.0 -> 19.1 us), at 32 11 %.
template <int DT, int KP, int NW, int ACT, bool TWICE>
__global__ __launch_bounds__(64 * NW, (FfnFused<DT, KP, NW>::WAVES)) void ffn_fused_kernel(const FfnParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
    using T = FfnType<DT>;
    using S = FfnFused<DT, KP, NW>;
    constexpr int E = T::E, NQ = T::NQ, RB = S::RB;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lh = lane >> 5;
    // this lane's pixel; found again after the loop rather than kept
    unsigned m, img;
    bool mine;
    unsigned long long at;
    auto place = [&](unsigned thread) {
        m = (blockIdx.x * NW + wave) * 32 + (thread & 31);
        mine = m < p.m;
        if (!mine) m = p.m - 1;
        img = (__umulhi(m, p.hw_mul) + m) >> p.hw_shift;
        at = (unsigned long long)(m - img * p.hw) * 32 + ((thread >> 5) & 1) * 16;
    };
    place(threadIdx.x);
    const unsigned lane_rows = ffn_lane_rows<DT>(lane), lane_down = FfnDownTile<DT>::lane(lane);

    // chunks of 32 hidden units of this part
    const int chunks = (p.hidden + 31) / 32;
    const int first = (int)((unsigned)chunks * blockIdx.y / gridDim.y), last = (int)((unsigned)chunks * (blockIdx.y + 1) / gridDim.y);
    auto stage = [&](int chunk) { FfnStager<DT, KP, NW>(p, wave, ffn_here(lane)).run(p, chunk, smem + ((chunk - first) & 1) * S::SLOT, wave, lane); };
    stage(first);
    u32x4 x[KP];
    ffn_load_planes<KP>(x, p.x.ptr + (long long)img * p.x.img_stride_b + at, p.x.plane_stride_b, p.kp_c);
    // b_down behind the two slots, 64 floats per wave; the first part of the hidden units adds it
    if (wave < (RB + 1) / 2) {
        const float* b = blockIdx.y == 0 ? p.b_down : nullptr;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(ffn_rsrc(b, b ? p.c * 4u : 0u), (__attribute__((address_space(3))) void*)(smem + 2 * S::SLOT + wave * 256), 4,
                                                 (wave * 64 + lane) * 4, 0, 0, 0);
    }
    static_assert((RB + 1) / 2 <= NW, "");
    ffn_meet();
    f32x16 y[RB];
    ffn_start_down<DT, RB>(y, smem + 2 * S::SLOT, lh);

    for (int chunk = first; chunk < last; ++chunk) {
        if (chunk > first) ffn_meet();
        const char* lds = smem + ((chunk - first) & 1) * S::SLOT;
        f32x16 g, u;
        ffn_start<DT>(g, u, lds + S::STAGE, lds + S::STAGE + 256, lh);
        if (chunk + 1 < last) stage(chunk + 1);
        const unsigned slot = (unsigned)(lds - smem);
        ffn_products<DT, KP>(g, u, x, smem, ffn_here(lane_rows + slot), S::UP);
        FfnDown<DT, RB> down;
        const unsigned down_at = ffn_here(lane_down + slot + 2 * S::UP);
        down.start(smem, down_at);
        u32x4 h[NQ], rest[NQ];
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            float v[E];
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = ffn_act<DT, ACT>(g[n * E + e]) * u[n * E + e];
            h[n] = ffn_pack<DT>(v);
            if constexpr (TWICE) rest[n] = ffn_pack_rest<DT>(v, h[n]);
        }
        ffn_zero_beyond<NQ>(h, p.kp_h - chunk * NQ);
        down.run(y, h, smem, down_at);
        if constexpr (TWICE) {
            down.start(smem, down_at);
            down.run(y, rest, smem, down_at);
        }
    }

    place(ffn_here(threadIdx.x));
    if (p.part) {
#pragma unroll
        for (int k = 0; k < KP; ++k)
            if (k < p.kp_c && mine) ffn_store_part<DT>(p, blockIdx.y, k, m, lh, y[k / NQ], (k % NQ) * E);
        return;
    }
    ffn_finish_pixel<DT, KP, RB>(p, y, p.res.ptr ? p.res.ptr + (long long)img * p.res.img_stride_b + at : nullptr,
                                 p.out.ptr + (long long)img * p.out.img_stride_b + at, p.res_scale, mine);
#endif
}

#if defined(__HIP_DEVICE_COMPILE__)
// out = res + scale * (sum of the parts) for a 16-byte piece: half of a plane of pixel m of `pixels`
template <int DT>
__device__ __forceinline__ void ffn_join_piece(const float* part, int parts, int planes, unsigned pixels, unsigned plane, unsigned m, float scale, const TView& res,
                                               const TView& out, unsigned hw, unsigned hw_mul, unsigned hw_shift, unsigned half) {
    constexpr int E = FfnType<DT>::E;
    float v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = 0.f;
    const float* s = part + (((unsigned long long)plane * pixels + m) * 2 + half) * E;
    const unsigned long long each = (unsigned long long)planes * pixels * 2 * E;
#pragma unroll 4
    for (int k = 0; k < parts; ++k)
#pragma unroll
        for (int e = 0; e < E; e += 4) {
            const f32x4 a = *(const f32x4*)(s + k * each + e);
            v[e] += a[0]; v[e + 1] += a[1]; v[e + 2] += a[2]; v[e + 3] += a[3];
        }
    const unsigned img = (__umulhi(m, hw_mul) + m) >> hw_shift;
    const unsigned long long at = (unsigned long long)(m - img * hw) * 32 + half * 16;
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] *= scale;
    if (res.ptr) {
        float o[E];
        ffn_unpack<DT>(*(const u32x4*)(res.ptr + (long long)img * res.img_stride_b + (long long)plane * res.plane_stride_b + at), o);
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] += o[e];
    }
    *(u32x4*)(out.ptr + (long long)img * out.img_stride_b + (long long)plane * out.plane_stride_b + at) = ffn_pack<DT>(v);
}
#endif

// The forward pass's, one thread = one piece
template <int DT>
__global__ __launch_bounds__(256) void ffn_join_kernel(const FfnParams p, int parts) {
#if defined(__HIP_DEVICE_COMPILE__)
    const unsigned long long i = ((unsigned long long)blockIdx.x * 256 + threadIdx.x) >> 1;  // plane, pixel
    const unsigned plane = (unsigned)(i / p.m), m = (unsigned)(i - (unsigned long long)plane * p.m);
    if (plane < (unsigned)p.kp_c)
        ffn_join_piece<DT>(p.part, parts, p.kp_c, p.m, plane, m, p.res_scale, p.res, p.out, p.hw, p.hw_mul, p.hw_shift, threadIdx.x & 1);
#endif
}

// ---- backward: hidden values and their gradients, and the gradient of x, in one launch ------------------------------------
// As the forward form: a wave keeps x, dy and (WITH_DX) the gradient of x of its 32 pixels in registers and walks the hidden
// units in chunks of 32.  Five products per chunk from three weight tiles: gate, up (rows = hidden units), dh = w_down^T dy, and with the
// rounded dg, du straight from the accumulators dx += w_gate^T dg + w_up^T du.  The two transposed ones read the tiles in LDS
// through transposing reads (half types: ds_read_b64_tr_b16, f32: four 4-byte reads), so no matrix is ever transposed in memory.
// hid, dg, du go to the workspace for the weights' gradients.  With few pixels blockIdx.y splits the hidden units; the parts leave
// f32 partial sums of dx that ffn_finish_kernel adds in order.
// Bound by vector work (activation, its slope, packing, bias sums: some 540 instructions per chunk and wave against 20 multiplies at
// four planes) where there are few pixels, so one wave per SIMD: 36864 pixels, c 64, hidden 256, bf16, gelu: 31 us, 2.0 us a chunk
// for one wave, 1.4 us for each of two on a SIMD.  131072 pixels, c 256, hidden 1024, bf16 (no dx): 265 to 290 us = 780 to 710 TFLOP/s while writing
// 0.8 GB.  Dealing chunks evenly over the CUs, with dx in parts, gained 7 % at 288 tiles of pixels and lost as much from 400 on.
template <int DT, int KP, bool WITH_DX>
struct FfnBack {
    static constexpr int NW = KP > kFfnBackPlanes ? 8 : 4;
    using F = FfnFused<DT, KP, NW>;
    static constexpr int REGS = 2 * KP * 4 + (WITH_DX ? F::RB * 16 : 0) + 48 + 72;
    static constexpr int WAVES = REGS <= 128 ? 4 : REGS <= 168 ? 3 : REGS <= 256 || NW == 8 ? 2 : 1;
    static constexpr int LDS = 2 * F::SLOT + 2 * NW * 256;  // two stages, two rows of 64 sums per wave
};

#if defined(__HIP_DEVICE_COMPILE__)
// Transposing reads: in each 16-lane group lane i gives the address of 8 bytes of row i / 4 and receives element i of the four
// rows; two of them (lo and hi, the same constant offset added to both) make the eight reduction values of an operand row.  In
// assembly with their wait, because behind the builtin the compiler waits for every LDS-DMA in flight before the first such
// read, which would end the overlap of the next stage with this one.
__device__ __forceinline__ unsigned ffn_lds_address(const char* p) { return (unsigned)(size_t)(const __attribute__((address_space(3))) char*)p; }
__device__ __forceinline__ u32x4 ffn_pair(const u32x2& l, const u32x2& h) { return u32x4{l[0], l[1], h[0], h[1]}; }
template <int A0, int A1>
__device__ __forceinline__ void ffn_tr_read2(u32x4 (&v)[2], unsigned lo, unsigned hi) {
    u32x2 a, b, c, d;
    asm volatile("ds_read_b64_tr_b16 %0, %4 offset:%6\n\tds_read_b64_tr_b16 %1, %5 offset:%6\n\t"
                 "ds_read_b64_tr_b16 %2, %4 offset:%7\n\tds_read_b64_tr_b16 %3, %5 offset:%7\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(a), "=&v"(b), "=&v"(c), "=&v"(d) : "v"(lo), "v"(hi), "n"(A0), "n"(A1) : "memory");
    v[0] = ffn_pair(a, b);
    v[1] = ffn_pair(c, d);
}
template <int A0, int A1, int A2, int A3>
__device__ __forceinline__ void ffn_tr_read4(u32x4 (&v)[4], unsigned lo, unsigned hi) {
    u32x2 a, b, c, d, e, f, g, h;
    asm volatile("ds_read_b64_tr_b16 %0, %8 offset:%10\n\tds_read_b64_tr_b16 %1, %9 offset:%10\n\t"
                 "ds_read_b64_tr_b16 %2, %8 offset:%11\n\tds_read_b64_tr_b16 %3, %9 offset:%11\n\t"
                 "ds_read_b64_tr_b16 %4, %8 offset:%12\n\tds_read_b64_tr_b16 %5, %9 offset:%12\n\t"
                 "ds_read_b64_tr_b16 %6, %8 offset:%13\n\tds_read_b64_tr_b16 %7, %9 offset:%13\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(a), "=&v"(b), "=&v"(c), "=&v"(d), "=&v"(e), "=&v"(f), "=&v"(g), "=&v"(h)
                 : "v"(lo), "v"(hi), "n"(A0), "n"(A1), "n"(A2), "n"(A3) : "memory");
    v[0] = ffn_pair(a, b);
    v[1] = ffn_pair(c, d);
    v[2] = ffn_pair(e, f);
    v[3] = ffn_pair(g, h);
}
// N operands of w_down^T from plane K0: rows = the chunk's 32 hidden units, reduction = a plane of the channels each.  The 8-byte
// segments of a row are taken in the order 0, 2, 1, 3, which puts the rows in the order of ffn_row.
template <int DT, int K0, int N>
__device__ __forceinline__ void ffn_weights_down_t(u32x4 (&v)[N], const char* lds, int lane) {
    const int lh = lane >> 5;
    if constexpr (DT == SRMI_F32) {
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int c = 8 * (K0 + i) + 4 * lh + j;
                v[i][j] = *(const unsigned*)(lds + (8 * c + (((lane & 31) >> 2) ^ ffn_key(c))) * 16 + (lane & 3) * 4);
            }
    } else {
        const int c = 8 * lh + ((lane >> 2) & 3), s = ((lane & 1) << 1) | ((lane >> 1) & 1);
        const int piece = ((lane >> 4) & 1) * 2 + (s >> 1);
        const unsigned lo = ffn_lds_address(lds + (s & 1) * 8 + (4 * c + (piece ^ ((c >> 2) & 3))) * 16);
        const unsigned hi = ffn_lds_address(lds + (s & 1) * 8 + (4 * (c + 4) + (piece ^ (((c + 4) >> 2) & 3))) * 16);
        if constexpr (N == 4) ffn_tr_read4<K0 * 1024, (K0 + 1) * 1024, (K0 + 2) * 1024, (K0 + 3) * 1024>(v, lo, hi);
        else ffn_tr_read2<K0 * 1024, (K0 + 1) * 1024>(v, lo, hi);
    }
}
// The operands of w_gate^T and w_up^T (v[0..1], v[2..3]: planes 0 and 1, or for f32 N0 and N0 + 1, of the chunk's hidden units as
// reduction) with rows = the 32 channels of block RB.
template <int DT, int RB, int N0, int UP>
__device__ __forceinline__ void ffn_weights_up_t(u32x4 (&v)[4], const char* lds, int lane) {
    const int lh = lane >> 5;
    if constexpr (DT == SRMI_F32) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int h = 8 * (N0 + (i & 1)) + 4 * lh + j;
                v[i][j] = *(const unsigned*)(lds + (i >> 1) * UP + RB * 4096 + (8 * h + (((lane & 31) >> 2) ^ ffn_key(h))) * 16 + (lane & 3) * 4);
            }
    } else {
        const int h = 8 * lh + ((lane >> 2) & 3), s = ((lane & 1) << 1) | ((lane >> 1) & 1);
        const int piece = (RB & 1) * 4 + ((lane >> 4) & 1) * 2 + (s >> 1);
        const unsigned lo = ffn_lds_address(lds + (s & 1) * 8 + (8 * h + (piece ^ ffn_key(h))) * 16);
        const unsigned hi = ffn_lds_address(lds + (s & 1) * 8 + (8 * (h + 4) + (piece ^ ffn_key(h + 4))) * 16);
        constexpr int at = (RB >> 1) * 4096;
        ffn_tr_read4<at, at + 2048, at + UP, at + UP + 2048>(v, lo, hi);
    }
}

#endif

#if defined(__HIP_DEVICE_COMPILE__)
// The three products of a chunk from plane K on, four planes (two, if there are only two) at a time
template <int DT, int KP, int K>
__device__ __forceinline__ void ffn_back_products(f32x16& g, f32x16& u, f32x16& dh, const u32x4 (&x)[KP], const u32x4 (&dy)[KP], const char* smem, unsigned at,
                                                  unsigned up, const char* down, int lane) {
    if constexpr (K < KP) {
        constexpr int N = KP < 4 ? 2 : 4;
        u32x4 t[N], w[2][2];
        auto read = [&](int k) {
            w[k % 2][0] = ffn_weights(smem, at, k % 4, (k / 4) * 4096);
            w[k % 2][1] = ffn_weights(smem, at, k % 4, up + (k / 4) * 4096);
        };
        read(K);
        ffn_weights_down_t<DT, K, N>(t, down, lane);
#pragma unroll
        for (int k = 0; k < N; ++k) {
            if (k + 1 < N) read(K + k + 1);
            __builtin_amdgcn_sched_barrier(0);
            ffn_mma<DT>(dh, t[k], dy[K + k]);
            ffn_mma<DT>(g, w[(K + k) % 2][0], x[K + k]);
            ffn_mma<DT>(u, w[(K + k) % 2][1], x[K + k]);
            __builtin_amdgcn_sched_barrier(0);
        }
        ffn_back_products<DT, KP, K + N>(g, u, dh, x, dy, smem, at, up, down, lane);
    }
}
// dx += w_gate^T dg + w_up^T du from channel block R on
template <int DT, int RB, int UP, int R>
__device__ __forceinline__ void ffn_back_dx(f32x16 (&dx)[RB], const u32x4 (&dg)[FfnType<DT>::NQ], const u32x4 (&du)[FfnType<DT>::NQ], const char* lds, int lane) {
    if constexpr (R < RB) {
        u32x4 w[4];
        ffn_weights_up_t<DT, R, 0, UP>(w, lds, lane);
        ffn_mma<DT>(dx[R], w[0], dg[0]);
        ffn_mma<DT>(dx[R], w[1], dg[1]);
        ffn_mma<DT>(dx[R], w[2], du[0]);
        ffn_mma<DT>(dx[R], w[3], du[1]);
        if constexpr (FfnType<DT>::NQ == 4) {
            ffn_weights_up_t<DT, R, 2, UP>(w, lds, lane);
            ffn_mma<DT>(dx[R], w[0], dg[2]);
            ffn_mma<DT>(dx[R], w[1], dg[3]);
            ffn_mma<DT>(dx[R], w[2], du[2]);
            ffn_mma<DT>(dx[R], w[3], du[3]);
        }
        ffn_back_dx<DT, RB, UP, R + 1>(dx, dg, du, lds, lane);
    }
}
#endif

template <int DT, int KP, bool WITH_DX, int ACT>
__global__ __launch_bounds__((64 * FfnBack<DT, KP, WITH_DX>::NW), (FfnBack<DT, KP, WITH_DX>::WAVES)) void ffn_back_kernel(const FfnParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
    using T = FfnType<DT>;
    using B = FfnBack<DT, KP, WITH_DX>;
    using S = typename B::F;
    constexpr int E = T::E, NQ = T::NQ, RB = S::RB, NW = B::NW;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lh = lane >> 5;
    unsigned m = p.m0 + (blockIdx.x * NW + wave) * 32 + (lane & 31);
    const bool mine = m < p.m;
    if (!mine) m = p.m - 1;
    const unsigned img = (__umulhi(m, p.hw_mul) + m) >> p.hw_shift;
    const unsigned long long at = (unsigned long long)(m - img * p.hw) * 32 + lh * 16;
    const unsigned long long hidden_at = ffn_hidden_pixel(m - p.m0, p.kp_h) + lh * 16;

    const int chunks = (p.hidden + 31) / 32;
    const int first = (int)((unsigned)chunks * blockIdx.y / gridDim.y), last = (int)((unsigned)chunks * (blockIdx.y + 1) / gridDim.y);
    auto stage = [&](int chunk) { FfnStager<DT, KP, NW>(p, wave, ffn_here(lane)).run(p, chunk, smem + (chunk & 1) * S::SLOT, wave, lane); };
    stage(first);
    u32x4 x[KP], dy[KP];  // zeros where the lane has no pixel, which keeps it out of the sums
    ffn_load_planes<KP>(x, p.x.ptr + (long long)img * p.x.img_stride_b + at, p.x.plane_stride_b, p.kp_c, mine);
    ffn_load_planes<KP>(dy, p.dy.ptr + (long long)img * p.dy.img_stride_b + at, p.dy.plane_stride_b, p.kp_c, mine);
    f32x16 dx[WITH_DX ? RB : 1];
#pragma unroll
    for (int r = 0; r < (WITH_DX ? RB : 1); ++r)
#pragma unroll
        for (int i = 0; i < 16; ++i) dx[r][i] = 0.f;
    const unsigned lane_rows = ffn_lane_rows<DT>(lane);
    float* red = (float*)(smem + 2 * S::SLOT);
    // the workgroup's bias sums of a chunk, one wave adds the waves' in order
    auto flush = [&](int chunk) {
        if (p.bias_part && wave == chunk % NW) {
            const float* r = red + (chunk & 1) * NW * 64 + lane;
            float s = r[0];
#pragma unroll
            for (int i = 1; i < NW; ++i) s += r[i * 64];
            const int ch = chunk * 32 + (lane & 31);
            if (ch < p.hidden) p.bias_part[((unsigned long long)blockIdx.x * 2 + lh) * p.hidden + ch] = s;
        }
    };

    // A chunk that is whole ends with 3 * NQ stores of each wave that has a pixel to store; the next chunk does not wait for them.
    const bool stores = __builtin_amdgcn_readfirstlane(__ballot(mine) != 0), full = __builtin_amdgcn_readfirstlane(__ballot(mine) == ~0ull);
    for (int chunk = first; chunk < last; ++chunk) {
        if (stores && chunk > first) ffn_meet_but<3 * NQ>();  // the chunk before was whole: only the last one can fall short
        else ffn_meet();
        const char* lds = smem + (chunk & 1) * S::SLOT;
        f32x16 g, u, dh;
        ffn_start<DT>(g, u, lds + S::STAGE, lds + S::STAGE + 256, lh);
#pragma unroll
        for (int i = 0; i < 16; ++i) dh[i] = 0.f;
        if (chunk > first) flush(chunk - 1);
        if (chunk + 1 < last) stage(chunk + 1);
        __builtin_amdgcn_sched_barrier(0);  // the stores below stay younger than the stage
        ffn_back_products<DT, KP, 0>(g, u, dh, x, dy, smem, ffn_here(lane_rows + (unsigned)(lds - smem)), S::UP, lds + 2 * S::UP, lane);
        float gv[16], uv[16];
        u32x4 dgf[NQ], duf[NQ];
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            float v[E];
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int i = n * E + e;
                float slope;
                const float a = ffn_act_slope<DT, ACT>(g[i], slope);
                const float d = p.res_scale * dh[i];
                v[e] = a * u[i];
                gv[i] = d * u[i] * slope;
                uv[i] = d * a;
            }
            dgf[n] = ffn_pack<DT>(gv + n * E);
            duf[n] = ffn_pack<DT>(uv + n * E);
            const int plane = chunk * NQ + n;
            if (mine && plane < p.kp_h) {
                const unsigned long long o = hidden_at + plane * kFfnHiddenPlane;
                *(u32x4*)(p.hid + o) = ffn_pack<DT>(v);
                *(u32x4*)(p.dg + o) = dgf[n];
                *(u32x4*)(p.du + o) = duf[n];
            }
        }
        if constexpr (WITH_DX) {
            ffn_zero_beyond<NQ>(dgf, p.kp_h - chunk * NQ);
            ffn_zero_beyond<NQ>(duf, p.kp_h - chunk * NQ);
            ffn_back_dx<DT, RB, S::UP, 0>(dx, dgf, duf, lds, lane);
        }
        if (p.bias_part) {
            if (!full) {  // an infinite weight or bias leaves NaN in lanes that have no pixel
#pragma unroll
                for (int i = 0; i < 16; ++i) { gv[i] = mine ? gv[i] : 0.f; uv[i] = mine ? uv[i] : 0.f; }
            }
            const float sg = ffn_spread_sums(gv, lane), su = ffn_spread_sums(uv, lane);
            // register i of half lh holds hidden unit CPB * (i / E) + E * lh + i % E of the chunk
            const int i = (lane >> 1) & 15, ch = T::CPB * (i / E) + E * lh + i % E;
            float* r = red + ((chunk & 1) * NW + wave) * 64;
            if (!(lane & 1)) { r[ch] = sg; r[32 + ch] = su; }
        }
    }
    if (p.bias_part) {
        __syncthreads();
        flush(last - 1);
    }
    if constexpr (WITH_DX) {
#pragma unroll
        for (int r = 0; r < RB; ++r)
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                const int plane = r * NQ + n;
                if (plane >= p.kp_c || !mine) continue;
                float v[E];
#pragma unroll
                for (int e = 0; e < E; ++e) v[e] = dx[r][n * E + e];
                if (p.part) {
                    ffn_store_part<DT>(p, blockIdx.y, plane, m, lh, dx[r], n * E);
                    continue;
                }
                *(u32x4*)(p.out.ptr + (long long)img * p.out.img_stride_b + plane * p.out.plane_stride_b + at) = ffn_pack<DT>(v);
            }
    }
#endif
}

// ---- weight gradients ------------------------------------------------------------------------------------------------------
// part[split] = sums over the split's pixels of dg[pixel][h] x[pixel][c], du x and hid dy (the last stored transposed, as
// w_down lies).  The reduction runs over pixels, so both operands are read from LDS transposed: half types with
// ds_read_b64_tr_b16, which hands a lane four pixels of one channel, f32 with four 4-byte reads.
// A workgroup of 8 waves takes 256 hidden units (4 x 64) x 32 * WJ * NJ channels; a wave's WJ = 4 gives 8 products for 6 operand
// reads.  With NJ = 1 the waves' other half takes every second operand of pixels; the two join in LDS at the end.  LDS holds
// four steps (f32: two) of 32 pixels, [plane][pixel][32 bytes], filled by LDS-DMA in pieces of 1 KiB (a step of a plane,
// contiguous in memory): one step is multiplied while the others are on their way, since a half-precision step's multiplies take less
// time than its loads.
// Planes are padded so that those of an operand lie in different banks.
// Measured: 131072 pixels, c 256, hidden 1024, bf16: 240 to 261 us = 860 to 790 TFLOP/s, 3.9 TB/s read; 36864 pixels, c 64, hidden 256: 16 us, 4 TB/s.
// One split of the pixels per CU (249 workgroups) and not two: the last step's partial sums are what a split costs.
template <int DT, int WJ, int NJ>
struct FfnWgrad {
    using T = FfnType<DT>;
    static constexpr int NW = 8, NK = kFfnWgradWaves / NJ;                 // waves, and how many of them share a tile of the output
    static constexpr int COLS = 32 * WJ * NJ;
    static constexpr int PU = 256 / T::CPB, PV = COLS / T::CPB;            // planes of the two sides
    static constexpr int STEP = 32;                                        // pixels
    static constexpr int PLANE = STEP * 32 + (DT == SRMI_F32 ? 64 : 128);  // bytes
    static constexpr int PIECES = (PU + PV + NW - 1) / NW;                 // of a wave (the last planes may be there for the count alone)
    static constexpr int SLOT = PIECES * NW * PLANE;
    static constexpr int SLOTS = DT == SRMI_F32 ? 2 : 4;
    static constexpr int LDS = SLOTS * SLOT;
};

#if defined(__HIP_DEVICE_COMPILE__)
// The operands of a multiply step: a[i] = 32 hidden units, b[j] = 32 channels (blocks of NQ planes from the two addresses), each x
// 16 bytes' worth of pixels from `pixel`.  Half types: a lane's four pixels of one channel per transposing read, all reads of
// a step in one block.
template <int DT, int PLANE, int WJ>
__device__ __forceinline__ void ffn_wgrad_operands(u32x4 (&a)[2], u32x4 (&b)[WJ], const char* u, const char* v, int pixel, int lane) {
    if constexpr (DT == SRMI_F32) {
        // multiply j takes pixels pixel + 2j + (lane / 32)
        const int at = ((lane & 31) >> 3) * PLANE + (pixel + (lane >> 5)) * 32 + (lane & 7) * 4;
        auto four = [](const char* s) { return u32x4{*(const unsigned*)s, *(const unsigned*)(s + 64), *(const unsigned*)(s + 128), *(const unsigned*)(s + 192)}; };
#pragma unroll
        for (int i = 0; i < 2; ++i) a[i] = four(u + at + i * 4 * PLANE);
#pragma unroll
        for (int j = 0; j < WJ; ++j) b[j] = four(v + at + j * 4 * PLANE);
    } else {
        const int at = ((lane >> 4) & 1) * PLANE + (pixel + 8 * (lane >> 5)) * 32 + (lane & 15) * 8;
        const unsigned ua = ffn_lds_address(u + at), va = ffn_lds_address(v + at);
        u32x2 p[4], q[8];
#define SRMI_TR(D, A, O) "ds_read_b64_tr_b16 " D ", " A " offset:" O "\n\t"
        if constexpr (WJ == 1) {
            asm volatile(SRMI_TR("%0", "%6", "0") SRMI_TR("%1", "%6", "128") SRMI_TR("%2", "%6", "%8") SRMI_TR("%3", "%6", "%9")
                         SRMI_TR("%4", "%7", "0") SRMI_TR("%5", "%7", "128") "s_waitcnt lgkmcnt(0)"
                         : "=&v"(p[0]), "=&v"(p[1]), "=&v"(p[2]), "=&v"(p[3]), "=&v"(q[0]), "=&v"(q[1])
                         : "v"(ua), "v"(va), "n"(2 * PLANE), "n"(2 * PLANE + 128) : "memory");
        } else if constexpr (WJ == 2) {
            asm volatile(SRMI_TR("%0", "%8", "0") SRMI_TR("%1", "%8", "128") SRMI_TR("%2", "%8", "%10") SRMI_TR("%3", "%8", "%11")
                         SRMI_TR("%4", "%9", "0") SRMI_TR("%5", "%9", "128") SRMI_TR("%6", "%9", "%10") SRMI_TR("%7", "%9", "%11") "s_waitcnt lgkmcnt(0)"
                         : "=&v"(p[0]), "=&v"(p[1]), "=&v"(p[2]), "=&v"(p[3]), "=&v"(q[0]), "=&v"(q[1]), "=&v"(q[2]), "=&v"(q[3])
                         : "v"(ua), "v"(va), "n"(2 * PLANE), "n"(2 * PLANE + 128) : "memory");
        } else if constexpr (WJ == 3) {
            asm volatile(SRMI_TR("%0", "%10", "0") SRMI_TR("%1", "%10", "128") SRMI_TR("%2", "%10", "%12") SRMI_TR("%3", "%10", "%13")
                         SRMI_TR("%4", "%11", "0") SRMI_TR("%5", "%11", "128") SRMI_TR("%6", "%11", "%12") SRMI_TR("%7", "%11", "%13")
                         SRMI_TR("%8", "%11", "%14") SRMI_TR("%9", "%11", "%15") "s_waitcnt lgkmcnt(0)"
                         : "=&v"(p[0]), "=&v"(p[1]), "=&v"(p[2]), "=&v"(p[3]), "=&v"(q[0]), "=&v"(q[1]), "=&v"(q[2]), "=&v"(q[3]), "=&v"(q[4]), "=&v"(q[5])
                         : "v"(ua), "v"(va), "n"(2 * PLANE), "n"(2 * PLANE + 128), "n"(4 * PLANE), "n"(4 * PLANE + 128) : "memory");
        } else {
            asm volatile(SRMI_TR("%0", "%12", "0") SRMI_TR("%1", "%12", "128") SRMI_TR("%2", "%12", "%14") SRMI_TR("%3", "%12", "%15")
                         SRMI_TR("%4", "%13", "0") SRMI_TR("%5", "%13", "128") SRMI_TR("%6", "%13", "%14") SRMI_TR("%7", "%13", "%15")
                         SRMI_TR("%8", "%13", "%16") SRMI_TR("%9", "%13", "%17") SRMI_TR("%10", "%13", "%18") SRMI_TR("%11", "%13", "%19") "s_waitcnt lgkmcnt(0)"
                         : "=&v"(p[0]), "=&v"(p[1]), "=&v"(p[2]), "=&v"(p[3]), "=&v"(q[0]), "=&v"(q[1]), "=&v"(q[2]), "=&v"(q[3]), "=&v"(q[4]), "=&v"(q[5]),
                           "=&v"(q[6]), "=&v"(q[7])
                         : "v"(ua), "v"(va), "n"(2 * PLANE), "n"(2 * PLANE + 128), "n"(4 * PLANE), "n"(4 * PLANE + 128), "n"(6 * PLANE), "n"(6 * PLANE + 128) : "memory");
        }
#undef SRMI_TR
#pragma unroll
        for (int i = 0; i < 2; ++i) a[i] = ffn_pair(p[2 * i], p[2 * i + 1]);
#pragma unroll
        for (int j = 0; j < WJ; ++j) b[j] = ffn_pair(q[2 * j], q[2 * j + 1]);
    }
}
#endif

template <int DT, int WJ, int NJ>
__global__ __launch_bounds__((64 * FfnWgrad<DT, WJ, NJ>::NW), 2) void ffn_wgrad_kernel(const FfnParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
    using T = FfnType<DT>;
    using G = FfnWgrad<DT, WJ, NJ>;
    constexpr int NW = G::NW;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unsigned tc = (p.c + G::COLS - 1) / G::COLS, th = (p.hidden + 255) / 256;
    // Workgroups go to the 8 XCDs in turn; renumbered so that an XCD takes whole splits, whose tiles read the same pixels of x
    // (dy) through its L2
    const unsigned total = gridDim.x * gridDim.y, lin = blockIdx.x + gridDim.x * blockIdx.y;
    const unsigned xcd = lin & 7u, q8 = total >> 3, r8 = total & 7u;
    const unsigned id = xcd * q8 + (xcd < r8 ? xcd : r8) + (lin >> 3);
    const unsigned split = id / gridDim.x, all = id - split * gridDim.x;
    const unsigned which = all / (tc * th), tile = all - which * tc * th;  // 0: w_gate, 1: w_up, 2: w_down
    const unsigned h0 = tile / tc * 256, c0 = (tile - tile / tc * tc) * G::COLS;
    const unsigned first = p.m0 + split * p.split_pixels;
    const unsigned end = p.m - first < p.split_pixels ? p.m : first + p.split_pixels;
    const char* hid_side = which == 0 ? p.dg : which == 1 ? p.du : p.hid;
    const TView& t = which == 2 ? p.dy : p.x;

    // This lane's pixel and byte of a step.  Every wave issues the same number of pieces per step, so that waits can count them: planes
    // beyond the tensors read the last one, which only reaches sums that are never stored.
    const unsigned px = lane >> 1;
    auto issue = [&](unsigned step, bool whole) {
        unsigned m = first + step * G::STEP + px;
        const bool mine = m < end;
        if (!mine) m = end - 1;
        const unsigned img = (__umulhi(m, p.hw_mul) + m) >> p.hw_shift;
        const char* a = hid_side + ffn_hidden_pixel(m - p.m0, p.kp_h) + (lane & 1) * 16;
        const char* b = t.ptr + (long long)img * t.img_stride_b + (unsigned long long)(m - img * p.hw) * 32 + (lane & 1) * 16;
        char* slot = smem + (step % G::SLOTS) * G::SLOT;
#pragma unroll
        for (int i = 0; i < G::PIECES; ++i) {
            const int plane = wave + NW * i;
            char* dst = slot + plane * G::PLANE;
            const bool u = plane < G::PU;
            const int q = u ? min((int)(h0 / T::CPB) + plane, p.kp_h - 1) : min((int)(c0 / T::CPB) + plane - G::PU, p.kp_c - 1);
            const char* src = u ? a + q * kFfnHiddenPlane : b + q * t.plane_stride_b;
            if (whole) {
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src, (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
            } else {  // the split's last step: pixels beyond it are zeros
                const u32x4 v = *(const u32x4*)src;
                *(u32x4*)(dst + lane * 16) = mine ? v : u32x4{0u, 0u, 0u, 0u};
            }
        }
    };

    f32x16 acc[2][WJ], ones_acc[WJ];
#pragma unroll
    for (int j = 0; j < WJ; ++j)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[0][j][i] = acc[1][j][i] = ones_acc[j][i] = 0.f;
    const int wi = wave % 4, wj = NJ == 2 ? wave / 4 : 0, wk = G::NK == 2 ? wave / 4 : 0;
    // the sums of dy (b_down's gradient) are products with ones, exact in f32; the four waves of a column take every fourth operand
    const bool dbias = which == 2 && h0 == 0 && p.db_part;
    u32x4 ones;
    if constexpr (DT == SRMI_F32) ones = u32x4{0x3f800000u, 0x3f800000u, 0x3f800000u, 0x3f800000u};
    else if constexpr (DT == SRMI_F16) ones = u32x4{0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u};
    else ones = u32x4{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};

    const unsigned whole = (end - first) / G::STEP, steps = (end - first + G::STEP - 1) / G::STEP;
#pragma unroll
    for (unsigned s = 0; s < G::SLOTS - 1; ++s)
        if (s < steps) issue(s, s < whole);
    for (unsigned s = 0; s < steps; ++s) {
        if (s + G::SLOTS - 2 < whole) ffn_meet_but<(G::SLOTS - 2) * G::PIECES>();
        else ffn_meet();
        if (s + G::SLOTS - 1 < steps) issue(s + G::SLOTS - 1, s + G::SLOTS - 1 < whole);
        const char* side = smem + (s % G::SLOTS) * G::SLOT;
        constexpr int KP = DT == SRMI_F32 ? 8 : 16;          // pixels of an operand
        constexpr int KS = G::STEP / KP / G::NK;              // operands of a wave in a step
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            const int pixel = (k * G::NK + wk) * KP;
            u32x4 a[2], b[WJ];
            ffn_wgrad_operands<DT, G::PLANE, WJ>(a, b, side + wi * 2 * T::NQ * G::PLANE, side + (G::PU + wj * WJ * T::NQ) * G::PLANE, pixel, lane);
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < WJ; ++j) ffn_mma<DT>(acc[i][j], a[i], b[j]);
            if (dbias && ((s * KS + k) & 3) == (unsigned)wi) {
#pragma unroll
                for (int j = 0; j < WJ; ++j) ffn_mma<DT>(ones_acc[j], ones, b[j]);
            }
        }
    }
    if constexpr (G::NK == 2) {
        // the second half of the waves hands its sums over through LDS, 32 hidden units at a time
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            f32x4* const mine = (f32x4*)smem + wi * WJ * 4 * 64 + lane;
            __syncthreads();
            if (wk == 1) {
#pragma unroll
                for (int j = 0; j < WJ; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) mine[(j * 4 + r) * 64] = f32x4{acc[i][j][4 * r], acc[i][j][4 * r + 1], acc[i][j][4 * r + 2], acc[i][j][4 * r + 3]};
            }
            __syncthreads();
            if (wk == 0) {
#pragma unroll
                for (int j = 0; j < WJ; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const f32x4 v = mine[(j * 4 + r) * 64];
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[i][j][4 * r + e] += v[e];
                    }
            }
        }
    }
    const int lh = lane >> 5;
    float* out = p.wpart + ((unsigned long long)split * 3 + which) * p.hidden * p.c;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < WJ; ++j) {
            const unsigned col = c0 + (wj * WJ + j) * 32 + (lane & 31);
            if (col >= (unsigned)p.c || wk) continue;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const unsigned row = h0 + (wi * 2 + i) * 32 + 8 * r + 4 * lh;  // hidden is a multiple of 8
                if (row >= (unsigned)p.hidden) continue;
                if (which == 2) {
                    *(f32x4*)(out + (unsigned long long)col * p.hidden + row) = f32x4{acc[i][j][4 * r], acc[i][j][4 * r + 1], acc[i][j][4 * r + 2], acc[i][j][4 * r + 3]};
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) out[(unsigned long long)(row + e) * p.c + col] = acc[i][j][4 * r + e];
                }
            }
        }
    if (dbias && lh == 0) {
#pragma unroll
        for (int j = 0; j < WJ; ++j) {
            const unsigned col = c0 + (wj * WJ + j) * 32 + lane;
            if (col < (unsigned)p.c) p.db_part[(((unsigned long long)split * G::NK + wk) * 4 + wi) * p.c + col] = ones_acc[j][0];
        }
    }
#endif
}

// ---- small kernels of the backward pass --------------------------------------------------------------------------------------
// blockIdx.z: w_gate, w_up ([hidden][c] -> [c][hidden]), w_down ([c][hidden] -> [hidden][c])
template <typename E>
__global__ __launch_bounds__(256) void ffn_transpose_kernel(const E* w_gate, const E* w_up, const E* w_down, E* t_gate, E* t_up, E* t_down, int c, int hidden) {
    __shared__ E tile[32][33];
    const E* src = blockIdx.z == 0 ? w_gate : blockIdx.z == 1 ? w_up : w_down;
    E* dst = blockIdx.z == 0 ? t_gate : blockIdx.z == 1 ? t_up : t_down;
    const int rows = blockIdx.z == 2 ? c : hidden, cols = blockIdx.z == 2 ? hidden : c;
    // the grid covers ceil(hidden / 32) x ceil(c / 32) tiles
    const int tr = (blockIdx.z == 2 ? blockIdx.y : blockIdx.x) * 32, tc = (blockIdx.z == 2 ? blockIdx.x : blockIdx.y) * 32;
    const int lx = threadIdx.x & 31, ly = threadIdx.x >> 5;
#pragma unroll
    for (int i = 0; i < 32; i += 8)
        if (tr + ly + i < rows && tc + lx < cols) tile[ly + i][lx] = src[(long long)(tr + ly + i) * cols + tc + lx];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 32; i += 8)
        if (tc + ly + i < cols && tr + lx < rows) dst[(long long)(tc + ly + i) * rows + tr + lx] = tile[lx][ly + i];
}

// Sums of `each` rows at a time of the hidden biases' partial sums (a row per tile of pixels), which the next launch adds.  Where one
// workgroup per 32 columns added all rows, the backward pass of c 16, hidden 16, f16 took 80 us at 2^18 pixels (2048 rows) and 8.8 ms at 2^25,
// so 74 us and 6.5 ms.
static __global__ __launch_bounds__(256) void ffn_bias_fold_kernel(const float* src, float* dst, int cols, int rows, int each) {
    __shared__ double red[8][32];
    const int lx = threadIdx.x & 31, grp = threadIdx.x >> 5, col = blockIdx.x * 32 + lx;
    const int first = blockIdx.y * each, last = min(rows - first, each) + first;
    double s = 0.0;
    if (col < cols) {
#pragma unroll 8
        for (int k = first + grp; k < last; k += 8) s += src[(long long)k * cols + col];
    }
    red[grp][lx] = s;
    __syncthreads();
    if (grp == 0 && col < cols) {
#pragma unroll
        for (int k = 1; k < 8; ++k) s += red[k][lx];
        dst[(long long)blockIdx.y * cols + col] = (float)s;
    }
}

// The gradients of weights and biases from their partial sums, in one launch: blocks of 128 weight elements, then blocks of 32
// columns of the biases: eight groups of threads take every eighth row and meet in LDS, a fixed order.  Then blocks of 128 pixels of
// a plane of dx, where it comes in parts.  The biases' rows are added in 64 bits: there are as many as pixels make tiles, and with equal terms a chain
// of f32 sums errs by 1.6e-4 at 2^25 pixels.
template <int DT>
__global__ __launch_bounds__(256) void ffn_finish_kernel(const FfnFinish f) {
    using E = std::conditional_t<DT == SRMI_F32, float, std::conditional_t<DT == SRMI_F16, _Float16, __bf16>>;
    __shared__ f32x4 red[8][32];
    const int lx = threadIdx.x & 31, grp = threadIdx.x >> 5;
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    if (blockIdx.x < f.w_blocks) {
        const long long i = ((long long)blockIdx.x * 32 + lx) * 4;  // `each` is a multiple of 4
        const bool live = i < 3 * f.each;
        if (live) {
#pragma unroll 4
            for (int k = grp; k < f.splits; k += 8) s += *(const f32x4*)(f.wpart + k * 3 * f.each + i);
        }
        red[grp][lx] = s;
        __syncthreads();
        if (grp || !live) return;
#pragma unroll
        for (int k = 1; k < 8; ++k) s += red[k][lx];
        const int which = (int)(i / f.each);
        const float scale = which == 2 ? f.res_scale : 1.f;
        E* dst = (E*)(which == 0 ? f.g_gate : which == 1 ? f.g_up : f.g_down) + (i - which * f.each);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (DT == SRMI_F16) dst[j] = to_f16_sat_nan(scale * s[j]);
            else dst[j] = (E)(scale * s[j]);
        }
        return;
    }
    const unsigned b = blockIdx.x - f.w_blocks;
#if defined(__HIP_DEVICE_COMPILE__)
    if (b >= f.b_blocks) {
        const unsigned plane = (b - f.b_blocks) / f.p_blocks, m = ((b - f.b_blocks) - plane * f.p_blocks) * 128 + (threadIdx.x >> 1);
        if (m < f.m) ffn_join_piece<DT>(f.part, f.parts, f.kp_c, f.m, plane, m, 1.f, {}, f.dx, f.hw, f.hw_mul, f.hw_shift, threadIdx.x & 1);
        return;
    }
#endif
    const unsigned which = b < f.h_blocks ? 0 : b < 2 * f.h_blocks ? 1 : 2;
    const int cols = which == 2 ? f.c : f.hidden, col = (int)(b - which * f.h_blocks) * 32 + lx;
    float* dst = which == 0 ? f.db_gate : which == 1 ? f.db_up : f.db_down;
    if (!dst) return;
    const float* src = which == 2 ? f.db_part : f.bias_part + which * f.hidden;
    const int rows = which == 2 ? f.db_rows : f.bias_rows;
    const long long stride = which == 2 ? f.c : 2ll * f.hidden;
    double v = 0.0;
    if (col < cols) {
#pragma unroll 8
        for (int k = grp; k < rows; k += 8) v += src[k * stride + col];
    }
    *(double*)&red[grp][lx] = v;
    __syncthreads();
    if (grp == 0 && col < cols) {
#pragma unroll
        for (int k = 1; k < 8; ++k) v += *(const double*)&red[k][lx];
        dst[col] = (float)(which == 2 ? f.res_scale * v : v);
    }
}

// ---- launches (one set per compute type) ------------------------------------------------------------------------------------
// LDS beyond the default limit of 64 KiB is an attribute of each function and device: the most a CU has, set once.
template <void (*KERNEL)(FfnParams)>
int ffn_allow_lds(size_t bytes) {
    static std::atomic<unsigned long long> configured{0};
    if (bytes <= 64 * 1024) return 0;
    int dev = 0;
    SRMI_HIP(hipGetDevice(&dev));
    const bool tracked = dev >= 0 && dev < 64;
    if (!tracked || !(configured.load(std::memory_order_acquire) >> dev & 1ull)) {
        SRMI_HIP(hipFuncSetAttribute((const void*)KERNEL, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
        if (tracked) configured.fetch_or(1ull << dev, std::memory_order_release);
    }
    return 0;
}

template <int DT, int WHAT, int RB, int ACT>
int ffn_launch_gemm_one(const FfnParams& p, hipStream_t s) {
    using S = FfnShape<WHAT, RB>;
    const unsigned rows = WHAT == kFfnHidden || WHAT == kFfnHiddenGrad ? p.hidden : p.c;
    if (ffn_allow_lds<ffn_gemm_kernel<DT, WHAT, RB, ACT>>(2 * S::STAGE)) return -1;
    const dim3 grid((p.m - p.m0 + S::PIXELS - 1) / S::PIXELS, (rows + S::ROWS - 1) / S::ROWS, p.part && RB == 1 && (WHAT == kFfnDown || WHAT == kFfnInputGrad) ? p.parts : 1);
    hipLaunchKernelGGL((ffn_gemm_kernel<DT, WHAT, RB, ACT>), grid, dim3(64 * S::NW), 2 * S::STAGE, s, p);
    SRMI_HIP(hipGetLastError());
    return 0;
}
template <int DT, int WHAT, int RB>
int ffn_launch_gemm_act(const FfnParams& p, int act, hipStream_t s) {
    switch (act) {
        case SRMI_ACT_NONE: return ffn_launch_gemm_one<DT, WHAT, RB, SRMI_ACT_NONE>(p, s);
        case SRMI_ACT_RELU: return ffn_launch_gemm_one<DT, WHAT, RB, SRMI_ACT_RELU>(p, s);
        case SRMI_ACT_LRELU: return ffn_launch_gemm_one<DT, WHAT, RB, SRMI_ACT_LRELU>(p, s);
        case SRMI_ACT_SILU: return ffn_launch_gemm_one<DT, WHAT, RB, SRMI_ACT_SILU>(p, s);
        default: return ffn_launch_gemm_one<DT, WHAT, RB, SRMI_ACT_GELU>(p, s);
    }
}
// 32-row blocks of a workgroup's tile.  Tiles of few rows read the pixels' operand more often but spread over more CUs, so a launch
// takes the largest of its instances that still gives every CU a workgroup, or the smallest.  Of those that do the products with
// c rows take the one that overhangs c least, of equal ones the largest.  Forward at c 512, hidden 1024, bf16: 4096 pixels 64 us with
// the large tiles only, 32 us so; 16384 pixels 92 and 78 us; asking for two workgroups per CU 31 and 75 us, but 107 against 100 us
// backward at 4096.
template <int WHAT>
int ffn_row_blocks(const FfnParams& p) {
    const bool to_hidden = WHAT == kFfnHidden || WHAT == kFfnHiddenGrad;
    const unsigned rows = to_hidden ? p.hidden : p.c, tiles = (p.m - p.m0 + 255) / 256;
    auto of = [&](unsigned blocks) { return (rows + 32 * blocks - 1) / (32 * blocks); };
    auto fills = [&](unsigned blocks) { return tiles * of(blocks) >= 256; };
    if (to_hidden) {
        if (WHAT == kFfnHidden && fills(4)) return 4;
    } else {
        const unsigned best = of(8) * 8 <= of(6) * 6 && of(8) * 8 <= of(4) * 4 ? 8 : of(6) * 6 <= of(4) * 4 ? 6 : 4;
        if (fills(best)) return best;
        if (fills(4)) return 4;
    }
    return fills(2) ? 2 : 1;
}
template <int DT, int WHAT>
int ffn_launch_gemm_rows(const FfnParams& p, hipStream_t s) {
    switch (ffn_row_blocks<WHAT>(p)) {
        case 8: return ffn_launch_gemm_one<DT, WHAT, 8, SRMI_ACT_NONE>(p, s);
        case 6: return ffn_launch_gemm_one<DT, WHAT, 6, SRMI_ACT_NONE>(p, s);
        case 4: return ffn_launch_gemm_one<DT, WHAT, 4, SRMI_ACT_NONE>(p, s);
        case 2: return ffn_launch_gemm_one<DT, WHAT, 2, SRMI_ACT_NONE>(p, s);
        default: return ffn_launch_gemm_one<DT, WHAT, 1, SRMI_ACT_NONE>(p, s);
    }
}
template <int DT>
int ffn_launch_any(const FfnParams& p, int what, int act, hipStream_t s) {
    if (what == kFfnHidden) {
        const int blocks = ffn_row_blocks<kFfnHidden>(p);
        return blocks == 4 ? ffn_launch_gemm_act<DT, kFfnHidden, 4>(p, act, s)
               : blocks == 2 ? ffn_launch_gemm_act<DT, kFfnHidden, 2>(p, act, s) : ffn_launch_gemm_act<DT, kFfnHidden, 1>(p, act, s);
    }
    if (what == kFfnDown) return ffn_launch_gemm_rows<DT, kFfnDown>(p, s);
    if (what == kFfnHiddenGrad)
        return ffn_row_blocks<kFfnHiddenGrad>(p) == 2 ? ffn_launch_gemm_act<DT, kFfnHiddenGrad, 2>(p, act, s) : ffn_launch_gemm_act<DT, kFfnHiddenGrad, 1>(p, act, s);
    return ffn_launch_gemm_rows<DT, kFfnInputGrad>(p, s);
}

template <int DT, int KP, int NW, int ACT, bool TWICE>
int ffn_launch_fused_one(const FfnParams& p, unsigned parts, hipStream_t s) {
    using S = FfnFused<DT, KP, NW>;
    constexpr size_t lds = 2 * S::SLOT + (S::RB + 1) / 2 * 256;
    if (ffn_allow_lds<ffn_fused_kernel<DT, KP, NW, ACT, TWICE>>(lds)) return -1;
    const dim3 grid((p.m + S::PIXELS - 1) / S::PIXELS, parts);
    hipLaunchKernelGGL((ffn_fused_kernel<DT, KP, NW, ACT, TWICE>), grid, dim3(64 * NW), lds, s, p);
    SRMI_HIP(hipGetLastError());
    return 0;
}
template <int DT, int KP, int NW, bool TWICE>
int ffn_launch_fused_act(const FfnParams& p, unsigned parts, int act, hipStream_t s) {
    switch (act) {
        case SRMI_ACT_NONE: return ffn_launch_fused_one<DT, KP, NW, SRMI_ACT_NONE, TWICE>(p, parts, s);
        case SRMI_ACT_RELU: return ffn_launch_fused_one<DT, KP, NW, SRMI_ACT_RELU, TWICE>(p, parts, s);
        case SRMI_ACT_LRELU: return ffn_launch_fused_one<DT, KP, NW, SRMI_ACT_LRELU, TWICE>(p, parts, s);
        case SRMI_ACT_SILU: return ffn_launch_fused_one<DT, KP, NW, SRMI_ACT_SILU, TWICE>(p, parts, s);
        default: return ffn_launch_fused_one<DT, KP, NW, SRMI_ACT_GELU, TWICE>(p, parts, s);
    }
}
template <int DT, int KP, int NW>
int ffn_launch_fused_pixels(const FfnParams& p, unsigned parts, int act, hipStream_t s) {
    const bool twice = DT != SRMI_F32 && p.m <= (unsigned)FfnFused<DT, KP, NW>::PIXELS;
    return twice ? ffn_launch_fused_act<DT, KP, NW, DT != SRMI_F32>(p, parts, act, s) : ffn_launch_fused_act<DT, KP, NW, false>(p, parts, act, s);
}
// The smallest instance whose KP planes hold the channels
template <int DT>
int ffn_launch_fused(const FfnParams& p, unsigned parts, int act, hipStream_t s) {
    if (p.kp_c <= 2) return ffn_launch_fused_pixels<DT, 2, 4>(p, parts, act, s);
    if (p.kp_c <= 4) return ffn_launch_fused_pixels<DT, 4, 4>(p, parts, act, s);
    if (p.kp_c <= 8) return ffn_launch_fused_pixels<DT, 8, 4>(p, parts, act, s);
    if (p.kp_c <= 12) return ffn_launch_fused_pixels<DT, 12, 4>(p, parts, act, s);
    return ffn_launch_fused_pixels<DT, 16, 8>(p, parts, act, s);
}

template <int DT, int KP, bool WITH_DX, int ACT>
int ffn_launch_back_one(const FfnParams& p, unsigned parts, hipStream_t s) {
    using B = FfnBack<DT, KP, WITH_DX>;
    if (ffn_allow_lds<ffn_back_kernel<DT, KP, WITH_DX, ACT>>(B::LDS)) return -1;
    hipLaunchKernelGGL((ffn_back_kernel<DT, KP, WITH_DX, ACT>), dim3((p.m - p.m0 + 32 * B::NW - 1) / (32 * B::NW), parts), dim3(64 * B::NW), B::LDS, s, p);
    SRMI_HIP(hipGetLastError());
    return 0;
}
template <int DT, int KP, bool WITH_DX>
int ffn_launch_back_act(const FfnParams& p, unsigned parts, int act, hipStream_t s) {
    switch (act) {
        case SRMI_ACT_NONE: return ffn_launch_back_one<DT, KP, WITH_DX, SRMI_ACT_NONE>(p, parts, s);
        case SRMI_ACT_RELU: return ffn_launch_back_one<DT, KP, WITH_DX, SRMI_ACT_RELU>(p, parts, s);
        case SRMI_ACT_LRELU: return ffn_launch_back_one<DT, KP, WITH_DX, SRMI_ACT_LRELU>(p, parts, s);
        case SRMI_ACT_SILU: return ffn_launch_back_one<DT, KP, WITH_DX, SRMI_ACT_SILU>(p, parts, s);
        default: return ffn_launch_back_one<DT, KP, WITH_DX, SRMI_ACT_GELU>(p, parts, s);
    }
}
// The gradient of x comes with it up to kFfnBackPlanes planes
template <int DT>
int ffn_launch_back(const FfnParams& p, unsigned parts, int act, hipStream_t s) {
    if (p.kp_c <= 2) return ffn_launch_back_act<DT, 2, true>(p, parts, act, s);
    if (p.kp_c <= 4) return ffn_launch_back_act<DT, 4, true>(p, parts, act, s);
    if (p.kp_c <= 8) return ffn_launch_back_act<DT, 8, true>(p, parts, act, s);
    if (p.kp_c <= 12) return ffn_launch_back_act<DT, 12, (kFfnBackPlanes >= 12)>(p, parts, act, s);
    return ffn_launch_back_act<DT, 16, false>(p, parts, act, s);
}

template <int DT>
int ffn_launch_join(const FfnParams& p, int parts, hipStream_t s) {
    const unsigned long long n = (unsigned long long)p.m * p.kp_c * 2;
    hipLaunchKernelGGL((ffn_join_kernel<DT>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, p, parts);
    SRMI_HIP(hipGetLastError());
    return 0;
}

template <int DT, int WJ, int NJ>
int ffn_launch_wgrad_one(const FfnParams& p, unsigned splits, hipStream_t s) {
    using G = FfnWgrad<DT, WJ, NJ>;
    if (ffn_allow_lds<ffn_wgrad_kernel<DT, WJ, NJ>>(G::LDS)) return -1;
    const unsigned tiles = 3u * ((p.c + G::COLS - 1) / G::COLS) * ((p.hidden + 255) / 256);
    hipLaunchKernelGGL((ffn_wgrad_kernel<DT, WJ, NJ>), dim3(tiles, splits), dim3(64 * G::NW), G::LDS, s, p);
    SRMI_HIP(hipGetLastError());
    return 0;
}
template <int DT>
int ffn_launch_wgrad(const FfnParams& p, unsigned splits, hipStream_t s) {
    switch (ffn_wgrad_cols(p.c)) {
        case 32: return ffn_launch_wgrad_one<DT, 1, 1>(p, splits, s);
        case 64: return ffn_launch_wgrad_one<DT, 2, 1>(p, splits, s);
        case 96: return ffn_launch_wgrad_one<DT, 3, 1>(p, splits, s);
        case 128: return ffn_launch_wgrad_one<DT, 4, 1>(p, splits, s);
        case 192: return ffn_launch_wgrad_one<DT, 3, 2>(p, splits, s);
        default: return ffn_launch_wgrad_one<DT, 4, 2>(p, splits, s);
    }
}

template <int DT>
int ffn_launch_finish(FfnFinish f, hipStream_t s) {
    if (f.fold) {
        const int rows = (f.bias_rows + f.fold - 1) / f.fold;
        hipLaunchKernelGGL(ffn_bias_fold_kernel, dim3((2 * f.hidden + 31) / 32, rows), dim3(256), 0, s, f.bias_part, f.bias_fold, 2 * f.hidden, f.bias_rows, f.fold);
        SRMI_HIP(hipGetLastError());
        f.bias_part = f.bias_fold;
        f.bias_rows = rows;
    }
    f.w_blocks = (unsigned)((3 * f.each / 4 + 31) / 32);
    f.h_blocks = (unsigned)((f.hidden + 31) / 32);
    f.b_blocks = f.db_down ? 2 * f.h_blocks + (f.c + 31) / 32 : f.db_gate || f.db_up ? 2 * f.h_blocks : 0;
    f.p_blocks = (f.m + 127) / 128;
    hipLaunchKernelGGL((ffn_finish_kernel<DT>), dim3(f.w_blocks + f.b_blocks + (f.part ? f.p_blocks * f.kp_c : 0)), dim3(256), 0, s, f);
    SRMI_HIP(hipGetLastError());
    return 0;
}

template <int DT>
int ffn_launch_transpose(const FfnParams& p, hipStream_t s) {
    using E = std::conditional_t<DT == SRMI_F32, unsigned, unsigned short>;
    hipLaunchKernelGGL((ffn_transpose_kernel<E>), dim3((p.hidden + 31) / 32, (p.c + 31) / 32, 3), dim3(256), 0, s, (const E*)p.w_gate, (const E*)p.w_up,
                       (const E*)p.w_down, (E*)p.wt_gate, (E*)p.wt_up, (E*)p.wt_down, p.c, p.hidden);
    SRMI_HIP(hipGetLastError());
    return 0;
}

template <int DT>
FfnLaunch ffn_launches() {
    return {ffn_launch_any<DT>, ffn_launch_fused<DT>, ffn_launch_join<DT>, ffn_launch_back<DT>, ffn_launch_wgrad<DT>, ffn_launch_finish<DT>, ffn_launch_transpose<DT>};
}

}  // namespace srmi
