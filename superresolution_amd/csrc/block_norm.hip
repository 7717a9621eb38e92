// The norms before and after a residual block, fused with the block's gate and residual scale, forward and backward:
//
//   v   = post ? norm(y) * post_weight + post_bias : y          norm over the channels of a pixel
//   sum = x + res_scale * gate[n][c] * v
//   out = norm(sum) * pre_weight + pre_bias                      the next block's input
//
// norm(v) = (v - mean) / sqrt(mean((v - mean)^2) + eps) (layer) or v / sqrt(mean(v^2) + eps) (rms).  All statistics are
// two-pass sums in f32 over values held in registers (a one-pass mean of squares loses the variance of channels whose mean is
// large against their spread); `out` is formed from the unrounded f32 sum.
//
// One pass over the data: a pixel's channels live in L lanes x NG granules of 8 channels, so both norms are register
// reductions plus log2(L) cross-lane steps, and x, y are read and sum, out written once.  The bound is HBM.
// Layout: a plane holds 32 bytes per pixel, so the two 16-byte halves of a half-precision plane go to neighbouring lanes,
// then the wave's 64 / L pixels, then the plane index: a wave reads (64 / L) * 32 contiguous bytes per plane.
// Measured: 8 x 256 x 256 pixels of 256 channels, bf16: 250 to 261 us = 4.3 to 4.1 TB/s, every byte moved once (a copy of 2 GiB: 4.9 TB/s); 339 x 510 x 64,
// f16 with an f32 trunk: 34 us = 3.9 TB/s; 32 vectors: 5 us, a launch.
#include "common.h"
#include "devutil.h"

namespace srmi {

struct NormParams {
    unsigned m;                   // pixels of all images
    unsigned hw, hw_mul, hw_shift;  // pixels of an image, and the reciprocal that divides by it
    int granules;                 // c / 8
    int c;
    int layer;
    float eps, inv_c, res_scale;
    int gate_stride;              // floats between the gate vectors of two images (0: one for all)
    TView x, y, sum, out;
    const float *post_w, *post_b, *pre_w, *pre_b, *gate;
    // backward
    TView d_sum, d_out, dx, dy;
    float* part;                  // [workgroup][kinds][c]
    float* gate_part;             // [n][chunks][c]
    unsigned n, chunks, seg;      // images; workgroups per image; pixels of a workgroup (flat form: of all images)
    int per_image;                // the gate has a vector per image: workgroups stay inside images
    int kinds;
};

// ---- accessors with the type fixed at compile time ---------------------------------------------------------------------
template <int DT>
__device__ __forceinline__ void get8(const TView& t, unsigned img, unsigned pix, int g, float (&v)[8]) {
    const char* a = t.ptr + (long long)img * t.img_stride_b + (unsigned long long)pix * 32;
    if constexpr (DT == SRMI_F32) {
        a += (long long)g * t.plane_stride_b;
        const f32x4 u = *(const f32x4*)a, w = *(const f32x4*)(a + 16);
#pragma unroll
        for (int j = 0; j < 4; ++j) { v[j] = u[j]; v[4 + j] = w[j]; }
    } else {
        a += (long long)(g >> 1) * t.plane_stride_b + (g & 1) * 16;
        if constexpr (DT == SRMI_F16) {
            const f16x8 u = *(const f16x8*)a;
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = (float)u[j];
        } else {
            const bf16x8 u = *(const bf16x8*)a;
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = (float)u[j];
        }
    }
}

template <int DT>
__device__ __forceinline__ void put8(const TView& t, unsigned img, unsigned pix, int g, const float (&v)[8]) {
    char* a = t.ptr + (long long)img * t.img_stride_b + (unsigned long long)pix * 32;
    if constexpr (DT == SRMI_F32) {
        a += (long long)g * t.plane_stride_b;
        *(f32x4*)a = f32x4{v[0], v[1], v[2], v[3]};
        *(f32x4*)(a + 16) = f32x4{v[4], v[5], v[6], v[7]};
    } else {
        a += (long long)(g >> 1) * t.plane_stride_b + (g & 1) * 16;
        if constexpr (DT == SRMI_F16) {
            f16x8 u;
#pragma unroll
            for (int j = 0; j < 8; ++j) u[j] = to_f16_sat_nan(v[j]);
            *(f16x8*)a = u;
        } else {
            bf16x8 u;
#pragma unroll
            for (int j = 0; j < 8; ++j) u[j] = (__bf16)v[j];
            *(bf16x8*)a = u;
        }
    }
}

// 8 floats of a per-channel vector; the caller's pointer need only be aligned to a float
typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));
__device__ __forceinline__ void vec8(const float* p, float (&v)[8]) {
    const f32x4_u a = *(const f32x4_u*)p, b = *(const f32x4_u*)(p + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) { v[j] = a[j]; v[4 + j] = b[j]; }
}

template <int CTRL>
__device__ __forceinline__ float dpp_get(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false));
}

// Sum over the L lanes that share a pixel (lane bit 0 and the bits above the pixel's), in every one of them.  Vector-pipe
// moves only (row swaps, rotations and a quad permute); each step adds the same two values on both sides, so all lanes
// get the same bits.
template <int L>
__device__ __forceinline__ float pixel_sum(float v) {
    if constexpr (L >= 4) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    if constexpr (L >= 8) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    if constexpr (L >= 16) v += dpp_get<0x128>(v);  // row_ror:8
    if constexpr (L >= 32) v += dpp_get<0x124>(v);  // row_ror:4: lanes 8 apart already agree
    if constexpr (L >= 64) v += dpp_get<0x4e>(v);   // quad_perm [2,3,0,1]
    return v + dpp_get<0xb1>(v);                    // quad_perm [1,0,3,2]
}

// The lane's place in its wave: which pixel, and which granules g = 2 * (hi + (L / 2) * j) + sub.
template <int L>
struct LaneMap {
    static constexpr int PW = 64 / L;  // pixels of a wave
    int pix, sub, hi;
    __device__ LaneMap() {
        const int lane = threadIdx.x & 63;
        sub = lane & 1;
        pix = (lane >> 1) & (PW - 1);
        hi = (lane >> 1) / PW;
    }
    __device__ int granule(int j) const { return 2 * (hi + (L / 2) * j) + sub; }
};

__device__ __forceinline__ void split_pixel(const NormParams& p, unsigned m, unsigned& img, unsigned& pix) {
    img = (__umulhi(m, p.hw_mul) + m) >> p.hw_shift;
    pix = m - img * p.hw;
}

// v -> its normalised form; returns 1 / std.  Only the last granule of a lane can lie beyond the last channel: `live` says
// whether it holds channels (its values are zero otherwise and stay so).
template <int L, int NG>
__device__ __forceinline__ float normalise(float (&v)[NG][8], const NormParams& p, bool live) {
    if (p.layer) {
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < NG; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) s += v[j][e];
        const float mean = pixel_sum<L>(s) * p.inv_c;
#pragma unroll
        for (int j = 0; j < NG; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[j][e] = j < NG - 1 || live ? v[j][e] - mean : 0.f;
    }
    float q = 0.f;
#pragma unroll
    for (int j = 0; j < NG; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) q += v[j][e] * v[j][e];
    const float r = 1.f / sqrtf(pixel_sum<L>(q) * p.inv_c + p.eps);
#pragma unroll
    for (int j = 0; j < NG; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[j][e] *= r;
    return r;
}

// DT: type of y and out; XT: type of x and sum (DT or f32)
template <int DT, int XT, int L, int NG>
__global__ __launch_bounds__(256) void block_norm_kernel(const NormParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
    const LaneMap<L> at;
    constexpr int PW = LaneMap<L>::PW;
    const unsigned stride = gridDim.x * 4u * PW;
    const bool live = at.granule(NG - 1) < p.granules;
    for (unsigned m0 = (blockIdx.x * 4u + (threadIdx.x >> 6)) * PW; m0 < p.m; m0 += stride) {
        const bool mine = m0 + at.pix < p.m;
        unsigned img, pix;
        split_pixel(p, mine ? m0 + at.pix : p.m - 1, img, pix);
        int g[NG];
#pragma unroll
        for (int j = 0; j < NG; ++j) g[j] = j < NG - 1 || live ? at.granule(j) : 0;
        float x[NG][8], v[NG][8];
#pragma unroll
        for (int j = 0; j < NG; ++j) get8<XT>(p.x, img, pix, g[j], x[j]);
        if (p.y.ptr) {
#pragma unroll
            for (int j = 0; j < NG; ++j) get8<DT>(p.y, img, pix, g[j], v[j]);
        }
        if (!live) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[NG - 1][e] = v[NG - 1][e] = 0.f;
        }
        if (p.y.ptr) {
            if (p.post_w) {
                normalise<L, NG>(v, p, live);
#pragma unroll
                for (int j = 0; j < NG; ++j) {
                    float w[8], b[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                    vec8(p.post_w + g[j] * 8, w);
                    if (p.post_b) vec8(p.post_b + g[j] * 8, b);
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[j][e] = v[j][e] * w[e] + b[e];
                }
            }
#pragma unroll
            for (int j = 0; j < NG; ++j) {
                float s[8];
                if (p.gate) {
                    vec8(p.gate + (unsigned long long)img * p.gate_stride + g[j] * 8, s);
#pragma unroll
                    for (int e = 0; e < 8; ++e) s[e] *= p.res_scale;
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) s[e] = p.res_scale;
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) x[j][e] += s[e] * v[j][e];
            }
            if (!live) {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[NG - 1][e] = 0.f;
            }
            if (p.sum.ptr && mine) {
#pragma unroll
                for (int j = 0; j < NG; ++j)
                    if (j < NG - 1 || live) put8<XT>(p.sum, img, pix, g[j], x[j]);
            }
        }
        if (p.out.ptr) {
            normalise<L, NG>(x, p, live);
#pragma unroll
            for (int j = 0; j < NG; ++j) {
                float w[8], b[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                vec8(p.pre_w + g[j] * 8, w);
                if (p.pre_b) vec8(p.pre_b + g[j] * 8, b);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[j][e] = x[j][e] * w[e] + b[e];
                if (mine && (j < NG - 1 || live)) put8<DT>(p.out, img, pix, g[j], x[j]);
            }
        }
    }
#endif
}

// ------------------------------------------------------------------------------------------------------------------------
// Backward.  With hat = normalised values, r = 1 / std, D = d_out * pre_weight and <.> the mean over a pixel's channels:
//   ds = d_sum + r_s * (D - <D * hat_s> * hat_s - [layer] <D>)       dx = ds
//   dv = res_scale * gate * ds                                        d_gate = res_scale * sum ds * v
//   d_post_weight = sum dv * hat_y   d_post_bias = sum dv             d_pre_weight = sum d_out * hat_s   d_pre_bias = sum d_out
//   dy = post ? r_y * (E - <E * hat_y> * hat_y - [layer] <E>), E = dv * post_weight : dv
// Statistics are recomputed from x and y.  The sums over pixels: a lane keeps its channels' sums in f32 registers over all
// pixels of its workgroup, the workgroup's lanes and waves join in LDS and write one row of partial sums, and a second
// kernel adds the rows: a fixed order throughout, no atomics.
// Measured: 4 x 256 x 256 pixels of 256 channels, f16 with an f32 trunk: 308 to 322 us = 3.9 to 3.75 TB/s, of which the second kernel 7; 16 x 48 x 48 x 64,
// bf16: 14 to 15 + 4 us; 4 x 256 x 256 x 64 in f32: 93 + 5 us (4.3 TB/s), forward 56 us (4.8).
// ------------------------------------------------------------------------------------------------------------------------
// Within an image res_scale * gate is a constant of the channel, so the lanes keep only A = sum ds * hat_y (or y) and B = sum ds for the
// three gradients behind the block: d_post_weight = res_scale * gate * A, d_post_bias = res_scale * gate * B, d_gate = res_scale *
// (post_weight * A + post_bias * B).
enum { kA = 0, kB = 1, kPreW = 2, kPreB = 3, kKinds = 4 };

// Adds over the lanes whose pixels differ in one bit of the lane number (mask M): with an even number N of values each half of the lanes keeps one
// half of the values, so that the work halves with every step; a single value both keep.
template <int M, int N>
__device__ __forceinline__ void pixel_fold(float (&v)[16], int lane) {
    constexpr bool HALVE = N % 2 == 0;
    constexpr int H = HALVE ? N / 2 : N;
    const bool up = lane & M;
#pragma unroll
    for (int i = 0; i < H; ++i) {
        const float lo = v[i], hi = HALVE ? v[i + H] : lo;
        if constexpr (M == 16 || M == 32) {
            const unsigned a = __float_as_uint(lo), b = __float_as_uint(hi);
            if constexpr (M == 16) {
                const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
                v[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
            } else {
                const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
                v[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
            }
        } else {
            // row_ror:12 brings lane + 4 to the lanes without the bit, row_ror:4 lane - 4 to those with it
            const float s = lo + (M == 2 ? dpp_get<0x4e>(lo) : M == 4 ? dpp_get<0x12c>(lo) : dpp_get<0x128>(lo));
            const float u = hi + (M == 2 ? dpp_get<0x4e>(hi) : M == 4 ? dpp_get<0x124>(hi) : dpp_get<0x128>(hi));
            v[i] = up ? u : s;
        }
    }
}

// Sums of a lane's NG * 8 channel values over the wave's pixels, spread over the lanes: afterwards the lane's first `left`
// values are those from index `first` on, and `owner` says whether it is the one to store them.
template <int L, int NG>
struct PixelFold {
    static constexpr int PW = 64 / L, BITS = PW == 32 ? 5 : PW == 16 ? 4 : PW == 8 ? 3 : PW == 4 ? 2 : PW == 2 ? 1 : 0;
    static constexpr int N = NG * 8, HALVINGS = NG == 1 ? 3 : 4;  // down to one value
    static constexpr int USED = BITS < HALVINGS ? BITS : HALVINGS, LEFT = N >> USED;
    static constexpr int at(int step) { return N >> (step < USED ? step : USED); }          // values before a step
    int first = 0;
    bool owner = true;
    __device__ explicit PixelFold(int lane) {
#pragma unroll
        for (int b = 0; b < BITS; ++b) {
            const int bit = (lane >> (b + 1)) & 1;
            if (b < USED) first += bit * (N >> (b + 1));
            else owner = owner && !bit;
        }
    }
    __device__ __forceinline__ void run(float (&v)[16], int lane) const {
        if constexpr (BITS > 0) pixel_fold<2, at(0)>(v, lane);
        if constexpr (BITS > 1) pixel_fold<4, at(1)>(v, lane);
        if constexpr (BITS > 2) pixel_fold<8, at(2)>(v, lane);
        if constexpr (BITS > 3) pixel_fold<16, at(3)>(v, lane);
        if constexpr (BITS > 4) pixel_fold<32, at(4)>(v, lane);
    }
};

// Joins one kind's sums over the lanes and waves of a workgroup and hands channel i's to take(i, sum), always in the same
// thread.  red: float[4][c] in LDS that nobody else touches until the next but one call.
template <int L, int NG, typename F>
__device__ __forceinline__ void join_sums(const float (&a)[NG][8], const LaneMap<L>& at, const NormParams& p, float* red, F take) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const PixelFold<L, NG> fold(lane);
    float v[16];
#pragma unroll
    for (int j = 0; j < NG; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[j * 8 + e] = a[j][e];
    fold.run(v, lane);
    if (fold.owner) {
#pragma unroll
        for (int i = 0; i < PixelFold<L, NG>::LEFT; ++i) {
            const int k = fold.first + i, g = at.granule(k >> 3);
            if (g < p.granules) red[wave * p.c + g * 8 + (k & 7)] = v[i];
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < p.c; i += 256) take(i, (red[i] + red[p.c + i]) + (red[2 * p.c + i] + red[3 * p.c + i]));
}

// A lane's share of a tensor as it lies in memory
template <int DT, int NG>
struct RawGranules {
    u32x4 v[NG][DT == SRMI_F32 ? 2 : 1];
    __device__ __forceinline__ void load(const TView& t, unsigned img, unsigned pix, const int (&g)[NG]) {
        const char* a = t.ptr + (long long)img * t.img_stride_b + (unsigned long long)pix * 32;
#pragma unroll
        for (int j = 0; j < NG; ++j) {
            if constexpr (DT == SRMI_F32) {
                v[j][0] = *(const u32x4*)(a + (long long)g[j] * t.plane_stride_b);
                v[j][DT == SRMI_F32 ? 1 : 0] = *(const u32x4*)(a + (long long)g[j] * t.plane_stride_b + 16);
            } else {
                v[j][0] = *(const u32x4*)(a + (long long)(g[j] >> 1) * t.plane_stride_b + (g[j] & 1) * 16);
            }
        }
    }
    // the values; those of the last granule are zeros where it lies beyond the last channel
    __device__ __forceinline__ void values(float (&f)[NG][8], bool live) const {
#pragma unroll
        for (int j = 0; j < NG; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if constexpr (DT == SRMI_F32) f[j][e] = __uint_as_float(v[j][e >> 2][e & 3]);
                else if constexpr (DT == SRMI_F16) f[j][e] = (float)__builtin_bit_cast(f16x8, v[j][0])[e];
                else f[j][e] = (float)__builtin_bit_cast(bf16x8, v[j][0])[e];
                if (j == NG - 1) f[j][e] = live ? f[j][e] : 0.f;
            }
    }
};

// 8 floats of a vector in LDS
__device__ __forceinline__ void lds8(const float* p, float (&v)[8]) {
    const f32x4 a = *(const f32x4*)p, b = *(const f32x4*)(p + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) { v[j] = a[j]; v[4 + j] = b[j]; }
}

// Per-channel vectors wait in LDS; the next pixels' tensors are requested before the present ones are worked on, since at three
// waves per SIMD (one granule of channels per lane; two, beyond 512 channels, leave one) little else hides the memory's latency.
template <int DT, int XT, int L, int NG>
__global__ __launch_bounds__(256, (NG == 1 ? 3 : 1)) void block_norm_backward_kernel(const NormParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
    extern __shared__ __attribute__((aligned(16))) float lds[];  // kNormLdsRows rows of c: vectors, then sums, then [2][4][c] joins
    float *const w_post = lds, *const b_post = lds + p.c, *const scale = lds + 2 * p.c, *const w_pre = lds + 3 * p.c;
    float *const total_a = lds + 4 * p.c, *const post_w = lds + 5 * p.c, *const post_b = lds + 6 * p.c, *const red = lds + 7 * p.c;
    const LaneMap<L> at;
    constexpr int PW = LaneMap<L>::PW;
    const bool live = at.granule(NG - 1) < p.granules;
    for (int i = threadIdx.x; i < p.c; i += 256) {
        w_post[i] = p.post_w ? p.post_w[i] : 1.f;
        b_post[i] = p.post_b ? p.post_b[i] : 0.f;
        scale[i] = p.gate && !p.per_image ? p.res_scale * p.gate[i] : p.res_scale;
        w_pre[i] = p.pre_w ? p.pre_w[i] : 0.f;
        post_w[i] = post_b[i] = 0.f;
    }
    float sums[kKinds][NG][8];
#pragma unroll
    for (int j = 0; j < NG; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
            for (int k = 0; k < kKinds; ++k) sums[k][j][e] = 0.f;
    // the workgroup's pixels: a run of all pixels (flat form), a run inside one image, or several whole images
    unsigned i0 = 0, i1 = 1, first = 0;
    if (p.per_image) {
        if (p.chunks > 1) {
            i0 = blockIdx.x / p.chunks;
            i1 = i0 + 1;
            first = (blockIdx.x - i0 * p.chunks) * p.seg;
        } else {
            i0 = (unsigned)((unsigned long long)p.n * blockIdx.x / gridDim.x);
            i1 = (unsigned)((unsigned long long)p.n * (blockIdx.x + 1) / gridDim.x);
        }
    } else {
        first = blockIdx.x * p.seg;
    }
    int g[NG];
#pragma unroll
    for (int j = 0; j < NG; ++j) g[j] = j < NG - 1 || live ? at.granule(j) : 0;

    for (unsigned i = i0; i < i1; ++i) {
        if (p.per_image) {
            for (int k = threadIdx.x; k < p.c; k += 256) scale[k] = p.res_scale * p.gate[(unsigned long long)i * p.c + k];
        }
        __syncthreads();
        const unsigned base = p.per_image ? i * p.hw : 0u;
        const unsigned limit = p.per_image ? p.hw : p.m;
        const unsigned end = base + (p.seg < limit - min(first, limit) ? first + p.seg : limit);
        RawGranules<XT, NG> rx, rds;
        RawGranules<DT, NG> ry, rdo;
        unsigned img, pix;
        bool mine;
        auto request = [&](unsigned m0) {
            mine = m0 + at.pix < end;
            split_pixel(p, mine ? m0 + at.pix : end - 1, img, pix);
            rx.load(p.x, img, pix, g);
            if (p.y.ptr) ry.load(p.y, img, pix, g);
            if (p.d_out.ptr) rdo.load(p.d_out, img, pix, g);
            if (p.d_sum.ptr) rds.load(p.d_sum, img, pix, g);
        };
        unsigned m0 = base + first + (threadIdx.x >> 6) * PW;
        if (m0 < end) request(m0);
        for (; m0 < end; m0 += 4u * PW) {
            float s[NG][8], v[NG][8], d[NG][8], ds[NG][8];
            rx.values(s, live);
            if (p.y.ptr) ry.values(v, live);
            if (p.d_out.ptr) rdo.values(d, live);
            if (p.d_sum.ptr) {
                rds.values(ds, live);
            } else {
#pragma unroll
                for (int j = 0; j < NG; ++j)
#pragma unroll
                    for (int e = 0; e < 8; ++e) ds[j][e] = 0.f;
            }
            const bool here = mine;
            const unsigned here_img = img, here_pix = pix;
            if (m0 + 4u * PW < end) request(m0 + 4u * PW);
            // (a lane without a pixel of its own repeats the last one's and adds zeros to the sums)
            float ry_std = 0.f;
            if (p.y.ptr) {
                if (p.post_w) ry_std = normalise<L, NG>(v, p, live);
#pragma unroll
                for (int j = 0; j < NG; ++j) {
                    float w[8], b[8], q[8];
                    lds8(w_post + g[j] * 8, w);
                    lds8(b_post + g[j] * 8, b);
                    lds8(scale + g[j] * 8, q);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        s[j][e] += q[e] * (v[j][e] * w[e] + b[e]);
                        if (j == NG - 1) s[j][e] = live ? s[j][e] : 0.f;
                    }
                }
            }
            if (p.d_out.ptr) {
                const float rs = normalise<L, NG>(s, p, live);
                float dot = 0.f, tot = 0.f;
#pragma unroll
                for (int j = 0; j < NG; ++j) {
                    float w[8];
                    lds8(w_pre + g[j] * 8, w);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float k = here ? d[j][e] : 0.f;
                        sums[kPreW][j][e] += here ? k * s[j][e] : 0.f;
                        sums[kPreB][j][e] += k;
                        d[j][e] *= w[e];
                        dot += d[j][e] * s[j][e];
                        tot += d[j][e];
                    }
                }
                dot = pixel_sum<L>(dot) * p.inv_c;
                tot = p.layer ? pixel_sum<L>(tot) * p.inv_c : 0.f;
#pragma unroll
                for (int j = 0; j < NG; ++j)
#pragma unroll
                    for (int e = 0; e < 8; ++e) ds[j][e] += rs * (d[j][e] - dot * s[j][e] - tot);
            }
            if (here) {
#pragma unroll
                for (int j = 0; j < NG; ++j)
                    if (j < NG - 1 || live) put8<XT>(p.dx, here_img, here_pix, g[j], ds[j]);
            }
            if (p.y.ptr) {
                float dot = 0.f, tot = 0.f;
#pragma unroll
                for (int j = 0; j < NG; ++j) {
                    float w[8], q[8];
                    lds8(w_post + g[j] * 8, w);
                    lds8(scale + g[j] * 8, q);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float k = here ? ds[j][e] : 0.f;
                        sums[kA][j][e] += here ? k * v[j][e] : 0.f;
                        sums[kB][j][e] += k;
                        d[j][e] = j < NG - 1 || live ? (q[e] * ds[j][e]) * w[e] : 0.f;
                        dot += d[j][e] * v[j][e];
                        tot += d[j][e];
                    }
                }
                if (p.post_w) {
                    dot = pixel_sum<L>(dot) * p.inv_c;
                    tot = p.layer ? pixel_sum<L>(tot) * p.inv_c : 0.f;
#pragma unroll
                    for (int j = 0; j < NG; ++j)
#pragma unroll
                        for (int e = 0; e < 8; ++e) d[j][e] = ry_std * (d[j][e] - dot * v[j][e] - tot);
                }
                if (here) {
#pragma unroll
                    for (int j = 0; j < NG; ++j)
                        if (j < NG - 1 || live) put8<DT>(p.dy, here_img, here_pix, g[j], d[j]);
                }
            }
        }
        if (p.y.ptr) {
            const unsigned slot = p.chunks > 1 ? blockIdx.x : i;
            float* gate = p.per_image ? p.gate_part + (unsigned long long)slot * p.c : nullptr;
            join_sums<L, NG>(sums[kA], at, p, red, [&](int c, float a) { total_a[c] = a; });
            join_sums<L, NG>(sums[kB], at, p, red + 4 * p.c, [&](int c, float b) {
                const float a = total_a[c];
                post_w[c] += scale[c] * a;
                post_b[c] += scale[c] * b;
                if (gate) gate[c] = w_post[c] * a + b_post[c] * b;
                else total_a[c] = w_post[c] * a + b_post[c] * b;
            });
#pragma unroll
            for (int j = 0; j < NG; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) sums[kA][j][e] = sums[kB][j][e] = 0.f;
        }
    }
    float* row = p.part + (unsigned long long)blockIdx.x * p.kinds * p.c;
    int k = 0;
    auto copy = [&](const float* v) {  // every channel in the thread that summed it
        for (int i = threadIdx.x; i < p.c; i += 256) row[p.c * k + i] = v[i];
        ++k;
    };
    if (p.post_w) copy(post_w);
    if (p.post_b) copy(post_b);
    if (p.d_out.ptr) {
        join_sums<L, NG>(sums[kPreW], at, p, red, [&](int c, float s) { row[p.c * k + c] = s; });
        ++k;
        if (p.pre_b) {
            join_sums<L, NG>(sums[kPreB], at, p, red + 4 * p.c, [&](int c, float s) { row[p.c * k + c] = s; });
            ++k;
        }
    }
    if (p.gate && !p.per_image) copy(total_a);
#endif
}

// Column sums of partial rows, in a fixed order.  blockIdx.y: a kind of vector, then the images of a per-image gate, whose rows are
// their own.  32 columns x 32 groups of rows per workgroup.
struct RowSums {
    const float *part, *gate_part;
    unsigned rows, gate_rows;  // workgroups; workgroups of an image
    int c, kinds;
    float* dst[5];
    float scale[5];
    float *d_gate, gate_scale;
};
__global__ __launch_bounds__(1024) void row_sums_kernel(const RowSums p, unsigned first_image) {
    __shared__ float red[32][33];
    const int lx = threadIdx.x & 31, col = blockIdx.x * 32 + lx, grp = threadIdx.x >> 5, k = blockIdx.y;
    const bool image = k >= p.kinds;
    const unsigned long long img = first_image + (unsigned)(k - p.kinds);
    const float* src = image ? p.gate_part + img * p.gate_rows * p.c : p.part + (long long)k * p.c;
    const unsigned rows = image ? p.gate_rows : p.rows;
    const long long stride = image ? p.c : (long long)p.kinds * p.c;
    float s = 0.f;
    if (col < p.c) {
#pragma unroll 8
        for (unsigned r = grp; r < rows; r += 32) s += src[r * stride + col];
    }
    red[grp][lx] = s;
    __syncthreads();
    if (grp == 0 && col < p.c) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) t += red[i][lx];
        if (image) p.d_gate[img * p.c + col] = p.gate_scale * t;
        else p.dst[k][col] = p.scale[k] * t;
    }
}

// ---- host --------------------------------------------------------------------------------------------------------------
constexpr int kNormMaxC = 1024;
constexpr int kNormLdsRows = 15;

// L lanes x NG granules with the fewest idle slots; of equal ones the largest NG, which gives a wave the most contiguous pixels
static void norm_shape(int granules, int max_ng, int* lanes, int* ng) {
    int best = 1 << 30;
    for (int l = 2; l <= 64; l *= 2) {
        const int k = (granules + l - 1) / l;
        if (k > max_ng) continue;
        if (l * k < best) { best = l * k; *lanes = l; *ng = k; }
    }
}

static void set_division(NormParams& p) {
    unsigned l = 0;
    while (l < 31 && (1u << l) < p.hw) ++l;
    p.hw_shift = l;
    p.hw_mul = (unsigned)((((1ull << l) - p.hw) << 32) / p.hw + 1);
}

static bool aligned_view(const srmi_tensor_t& t) {
    const long long es = dtype_size(t.dtype);
    return (((uintptr_t)t.ptr | (unsigned long long)(t.img_stride * es) | (unsigned long long)(t.plane_stride * es)) & 15) == 0;
}

static bool float_type(int dt) { return dt == SRMI_F32 || dt == SRMI_F16 || dt == SRMI_BF16; }

// What both directions check; *dt / *xt: the two element types.
static int check_norm(const char* who, int n, int h, int w, int c, int kind, float eps, const srmi_tensor_t& x, const srmi_tensor_t& y,
                      const srmi_tensor_t* others[], int n_others, const bool trunk[], bool has_pre, const float* post_w, const float* post_b,
                      const float* pre_b, const float* gate, int* dt, int* xt) {
    if (n <= 0 || h <= 0 || w <= 0 || c <= 0 || c % 8 || c > kNormMaxC)
        SRMI_FAIL("%s: bad shape n=%d h=%d w=%d c=%d (c: a multiple of the plane width, at most %d)", who, n, h, w, c, kNormMaxC);
    if ((long long)n * h * w >= (1ll << 31)) SRMI_FAIL("%s: 2^31 pixels or more", who);
    if (kind != SRMI_NORM_LAYER && kind != SRMI_NORM_RMS) SRMI_FAIL("%s: kind must be SRMI_NORM_LAYER or SRMI_NORM_RMS", who);
    if (!(eps >= 0.f)) SRMI_FAIL("%s: eps must not be negative", who);
    if (!x.ptr) SRMI_FAIL("%s: no x", who);
    if (!y.ptr && (post_w || gate)) SRMI_FAIL("%s: a norm or a gate for a block output y that is not there", who);
    if (!y.ptr && !has_pre) SRMI_FAIL("%s: neither a block output y nor a norm before the next block", who);
    if (post_b && !post_w) SRMI_FAIL("%s: post_bias without post_weight", who);
    if (pre_b && !has_pre) SRMI_FAIL("%s: pre_bias without pre_weight", who);
    *xt = x.dtype;
    *dt = y.ptr ? y.dtype : -1;
    for (int i = 0; i < n_others; ++i) {
        const srmi_tensor_t& t = *others[i];
        if (!t.ptr) continue;
        if (trunk[i]) {
            if (t.dtype != *xt) SRMI_FAIL("%s: the tensors of the residual trunk must be of the type of x", who);
        } else {
            if (*dt >= 0 && t.dtype != *dt) SRMI_FAIL("%s: the tensors of the block must be of one type", who);
            *dt = t.dtype;
        }
        if (!aligned_view(t)) SRMI_FAIL("%s: tensor addresses and strides must be multiples of 16 bytes", who);
    }
    if (*dt < 0) *dt = *xt;
    if (!float_type(*dt) || !float_type(*xt)) SRMI_FAIL("%s: tensors must be f32, f16 or bf16", who);
    if (*xt != *dt && *xt != SRMI_F32) SRMI_FAIL("%s: x must be of the block's type or f32", who);
    if (c % dtype_cpb(*dt)) SRMI_FAIL("%s: c=%d is not a multiple of the plane width %d", who, c, dtype_cpb(*dt));
    if (!aligned_view(x) || (y.ptr && !aligned_view(y))) SRMI_FAIL("%s: tensor addresses and strides must be multiples of 16 bytes", who);
    return 0;
}

static void fill_common(NormParams& p, int n, int h, int w, int c, int kind, float eps, float res_scale, int gate_per_image) {
    p.n = (unsigned)n;
    p.hw = (unsigned)h * (unsigned)w;
    p.m = p.n * p.hw;
    set_division(p);
    p.c = c;
    p.granules = c / 8;
    p.layer = kind == SRMI_NORM_LAYER;
    p.eps = eps;
    p.inv_c = 1.f / (float)c;
    p.res_scale = res_scale;
    p.gate_stride = gate_per_image ? c : 0;
}

template <int DT, int XT, int L>
static void launch_forward(const NormParams& p, int ng, unsigned grid, hipStream_t s) {
    if (ng == 1) hipLaunchKernelGGL((block_norm_kernel<DT, XT, L, 1>), dim3(grid), dim3(256), 0, s, p);
    else if (ng == 2) hipLaunchKernelGGL((block_norm_kernel<DT, XT, L, 2>), dim3(grid), dim3(256), 0, s, p);
    else if (ng == 3) hipLaunchKernelGGL((block_norm_kernel<DT, XT, L, 3>), dim3(grid), dim3(256), 0, s, p);
    else hipLaunchKernelGGL((block_norm_kernel<DT, XT, L, 4>), dim3(grid), dim3(256), 0, s, p);
}

template <int DT, int XT, int L>
static void launch_backward(const NormParams& p, int ng, unsigned grid, hipStream_t s) {
    const size_t lds = (size_t)kNormLdsRows * p.c * sizeof(float);  // at most 60 KiB
    if (ng == 1) hipLaunchKernelGGL((block_norm_backward_kernel<DT, XT, L, 1>), dim3(grid), dim3(256), lds, s, p);
    else hipLaunchKernelGGL((block_norm_backward_kernel<DT, XT, L, 2>), dim3(grid), dim3(256), lds, s, p);
}

template <int DT, int XT, bool BACK>
static void launch_types(const NormParams& p, int lanes, int ng, unsigned grid, hipStream_t s) {
    switch (lanes) {
#define SRMI_NORM_LANES(L)                                          \
    case L:                                                         \
        if constexpr (BACK) launch_backward<DT, XT, L>(p, ng, grid, s); \
        else launch_forward<DT, XT, L>(p, ng, grid, s);             \
        break;
        SRMI_NORM_LANES(2)
        SRMI_NORM_LANES(4)
        SRMI_NORM_LANES(8)
        SRMI_NORM_LANES(16)
        SRMI_NORM_LANES(32)
        SRMI_NORM_LANES(64)
#undef SRMI_NORM_LANES
    }
}

template <bool BACK>
static void launch_norm(int dt, int xt, const NormParams& p, int lanes, int ng, unsigned grid, hipStream_t s) {
    if (dt == SRMI_F32) launch_types<SRMI_F32, SRMI_F32, BACK>(p, lanes, ng, grid, s);
    else if (dt == SRMI_F16 && xt == SRMI_F16) launch_types<SRMI_F16, SRMI_F16, BACK>(p, lanes, ng, grid, s);
    else if (dt == SRMI_F16) launch_types<SRMI_F16, SRMI_F32, BACK>(p, lanes, ng, grid, s);
    else if (xt == SRMI_BF16) launch_types<SRMI_BF16, SRMI_BF16, BACK>(p, lanes, ng, grid, s);
    else launch_types<SRMI_BF16, SRMI_F32, BACK>(p, lanes, ng, grid, s);
}

// The backward pass's split of the pixels over workgroups, a function of the shape alone (the workspace's size follows it).
struct NormSplit {
    unsigned grid, chunks, seg;
    int lanes, ng;
};
constexpr unsigned kNormWorkgroups = 768;  // three per CU, what the registers allow
static NormSplit norm_split(int n, long long hw, int c, bool per_image) {
    NormSplit s = {};
    // One granule per lane keeps three waves per SIMD; with two a wave touches half as many planes for the same bytes, which outweighs
    // that from 256 channels on where both shapes fill their lanes (4 x 256 x 256 at 256 channels: 322 against 433 us, 510 x 339
    // at 64: 59 against 47 us, at 192, which two per lane do not fill: 138 against 114 us).
    const bool full = c >= 256 && (c & (c - 1)) == 0;
    norm_shape(c / 8, c > 512 || full ? 2 : 1, &s.lanes, &s.ng);
    const unsigned step = 4u * (64u / (unsigned)s.lanes);  // pixels of a workgroup's iteration
    const unsigned long long span = per_image ? (unsigned long long)hw : (unsigned long long)n * hw;
    const unsigned want = per_image ? ((unsigned)n >= kNormWorkgroups ? 1u : kNormWorkgroups / (unsigned)n) : kNormWorkgroups;
    unsigned long long seg = (span + want - 1) / want;
    seg = (seg + step - 1) / step * step;
    if (seg < 2 * step) seg = 2 * step;  // the joins at its end take a workgroup as long as a few steps
    s.chunks = (unsigned)((span + seg - 1) / seg);
    s.seg = (unsigned)seg;
    if (!per_image) s.grid = s.chunks;
    else if (s.chunks > 1) s.grid = s.chunks * (unsigned)n;
    else s.grid = (unsigned)n < kNormWorkgroups ? (unsigned)n : kNormWorkgroups;
    return s;
}
static int norm_kinds(const srmi_block_norm_grad_desc_t* d, bool per_image) {
    return (d->post_weight ? 1 : 0) + (d->post_bias ? 1 : 0) + (d->pre_weight ? 1 : 0) + (d->pre_bias ? 1 : 0) + (d->gate && !per_image ? 1 : 0);
}

}  // namespace srmi

using namespace srmi;

extern "C" int srmi_block_norm(const srmi_block_norm_desc_t* d, void* hip_stream) {
    const char* who = "srmi_block_norm";
    if (!d) SRMI_FAIL("%s: null descriptor", who);
    const srmi_tensor_t* others[] = {&d->sum, &d->out};
    const bool trunk[] = {true, false};
    int dt, xt;
    if (check_norm(who, d->n, d->h, d->w, d->c, d->kind, d->eps, d->x, d->y, others, 2, trunk, d->pre_weight != nullptr, d->post_weight, d->post_bias,
                   d->pre_bias, d->gate, &dt, &xt))
        return -1;
    if ((d->pre_weight != nullptr) != (d->out.ptr != nullptr)) SRMI_FAIL("%s: out goes with pre_weight", who);
    if (d->sum.ptr && !d->y.ptr) SRMI_FAIL("%s: without y the sum is x", who);
    if (!d->sum.ptr && !d->out.ptr) SRMI_FAIL("%s: no output tensor", who);
    NormParams p = {};
    fill_common(p, d->n, d->h, d->w, d->c, d->kind, d->eps, d->res_scale, d->gate_per_image);
    p.x = to_view(d->x); p.y = to_view(d->y); p.sum = to_view(d->sum); p.out = to_view(d->out);
    p.post_w = d->post_weight; p.post_b = d->post_bias; p.pre_w = d->pre_weight; p.pre_b = d->pre_bias; p.gate = d->gate;
    int lanes = 0, ng = 0;
    norm_shape(p.granules, 4, &lanes, &ng);
    const unsigned step = 4u * (64u / (unsigned)lanes);
    const unsigned long long wg = ((unsigned long long)p.m + step - 1) / step;
    const unsigned grid = wg < 16384ull ? (unsigned)wg : 16384u;
    launch_norm<false>(dt, xt, p, lanes, ng, grid, (hipStream_t)hip_stream);
    SRMI_HIP(hipGetLastError());
    return 0;
}

extern "C" size_t srmi_block_norm_backward_workspace(const srmi_block_norm_grad_desc_t* d) {
    if (!d || d->n <= 0 || d->h <= 0 || d->w <= 0 || d->c <= 0 || d->c % 8 || d->c > kNormMaxC || (long long)d->n * d->h * d->w >= (1ll << 31)) return 0;
    const bool per_image = d->gate && d->gate_per_image;
    const NormSplit s = norm_split(d->n, (long long)d->h * d->w, d->c, per_image);
    size_t floats = (size_t)s.grid * norm_kinds(d, per_image) * d->c;
    if (per_image) floats += (size_t)d->n * s.chunks * d->c;
    return floats * sizeof(float);
}

extern "C" int srmi_block_norm_backward(const srmi_block_norm_grad_desc_t* d, void* workspace, size_t workspace_bytes, void* hip_stream) {
    const char* who = "srmi_block_norm_backward";
    if (!d) SRMI_FAIL("%s: null descriptor", who);
    const srmi_tensor_t* others[] = {&d->d_sum, &d->dx, &d->d_out, &d->dy};
    const bool trunk[] = {true, true, false, false};
    int dt, xt;
    if (check_norm(who, d->n, d->h, d->w, d->c, d->kind, d->eps, d->x, d->y, others, 4, trunk, d->pre_weight != nullptr, d->post_weight, d->post_bias,
                   d->pre_bias, d->gate, &dt, &xt))
        return -1;
    if ((d->pre_weight != nullptr) != (d->d_out.ptr != nullptr)) SRMI_FAIL("%s: d_out goes with pre_weight", who);
    if (!d->d_sum.ptr && !d->d_out.ptr) SRMI_FAIL("%s: neither d_sum nor d_out", who);
    if (!d->dx.ptr || (d->y.ptr != nullptr) != (d->dy.ptr != nullptr)) SRMI_FAIL("%s: dx, and dy with y, must be given", who);
    if ((d->gate != nullptr) != (d->d_gate != nullptr) || (d->post_weight != nullptr) != (d->d_post_weight != nullptr) ||
        (d->post_bias != nullptr) != (d->d_post_bias != nullptr) || (d->pre_weight != nullptr) != (d->d_pre_weight != nullptr) ||
        (d->pre_bias != nullptr) != (d->d_pre_bias != nullptr))
        SRMI_FAIL("%s: every gate, weight and bias comes with its gradient's place, and none without", who);
    const bool per_image = d->gate && d->gate_per_image;
    const size_t need = srmi_block_norm_backward_workspace(d);
    if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15)))
        SRMI_FAIL("%s: needs %zu bytes of workspace on a multiple of 16 (got %zu)", who, need, workspace ? workspace_bytes : (size_t)0);
    NormParams p = {};
    fill_common(p, d->n, d->h, d->w, d->c, d->kind, d->eps, d->res_scale, d->gate_per_image);
    p.x = to_view(d->x); p.y = to_view(d->y); p.d_sum = to_view(d->d_sum); p.d_out = to_view(d->d_out); p.dx = to_view(d->dx); p.dy = to_view(d->dy);
    p.post_w = d->post_weight; p.post_b = d->post_bias; p.pre_w = d->pre_weight; p.pre_b = d->pre_bias; p.gate = d->gate;
    const NormSplit sp = norm_split(d->n, (long long)d->h * d->w, d->c, per_image);
    p.per_image = per_image; p.chunks = sp.chunks; p.seg = sp.seg;
    p.kinds = norm_kinds(d, per_image);
    p.part = (float*)workspace;
    p.gate_part = per_image ? p.part + (size_t)sp.grid * p.kinds * p.c : nullptr;
    hipStream_t s = (hipStream_t)hip_stream;
    launch_norm<true>(dt, xt, p, sp.lanes, sp.ng, sp.grid, s);
    SRMI_HIP(hipGetLastError());
    RowSums r = {};
    r.part = p.part; r.rows = sp.grid; r.c = p.c;
    r.gate_part = p.gate_part; r.gate_rows = sp.chunks; r.d_gate = d->d_gate; r.gate_scale = d->res_scale;
    auto add = [&](float* dst, float scale) { if (dst) { r.dst[r.kinds] = dst; r.scale[r.kinds++] = scale; } };
    add(d->d_post_weight, 1.f); add(d->d_post_bias, 1.f); add(d->d_pre_weight, 1.f); add(d->d_pre_bias, 1.f);
    if (!per_image) add(d->d_gate, d->res_scale);
    const unsigned cols = (unsigned)(p.c + 31) / 32, images = per_image ? p.n : 0u;
    unsigned done = 0;
    do {  // a grid has at most 65535 rows
        const unsigned now = images - done < 65000u ? images - done : 65000u;
        if (r.kinds + now) hipLaunchKernelGGL(row_sums_kernel, dim3(cols, r.kinds + now), dim3(1024), 0, s, r, done);
        SRMI_HIP(hipGetLastError());
        done += now;
        r.kinds = 0;
    } while (done < images);
    return 0;
}
