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
#include "common.h"
#include "devutil.h"
#include "row_sums.h"

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
// ------------------------------------------------------------------------------------------------------------------------
enum { kPostW = 0, kPostB = 1, kPreW = 2, kPreB = 3, kKinds = 4 };

// Joins one kind's sums over the lanes and waves of a workgroup: dst[c].  red: float[4][c] in LDS.
template <int L, int NG>
__device__ __forceinline__ void join_sums(float (&a)[NG][8], const LaneMap<L>& at, const NormParams& p, bool live, float* red, float* dst) {
    constexpr int PW = LaneMap<L>::PW;
    const int wave = threadIdx.x >> 6;
#pragma unroll
    for (int j = 0; j < NG; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float s = a[j][e];
#pragma unroll
            for (int o = 2; o < 2 * PW; o <<= 1) s += __shfl_xor(s, o);
            a[j][e] = s;
        }
    if (at.pix == 0) {
#pragma unroll
        for (int j = 0; j < NG; ++j)
            if (j < NG - 1 || live) {
#pragma unroll
                for (int e = 0; e < 8; ++e) red[wave * p.c + at.granule(j) * 8 + e] = a[j][e];
            }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < p.c; i += 256) dst[i] = (red[i] + red[p.c + i]) + (red[2 * p.c + i] + red[3 * p.c + i]);
    __syncthreads();
}

template <int DT, int XT, int L, int NG>
__global__ __launch_bounds__(256) void block_norm_backward_kernel(const NormParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
    extern __shared__ float red[];  // [4][c]
    const LaneMap<L> at;
    constexpr int PW = LaneMap<L>::PW;
    const bool live = at.granule(NG - 1) < p.granules;
    float sums[kKinds][NG][8], gsum[NG][8];
#pragma unroll
    for (int j = 0; j < NG; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            gsum[j][e] = 0.f;
#pragma unroll
            for (int k = 0; k < kKinds; ++k) sums[k][j][e] = 0.f;
        }
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
        const unsigned base = p.per_image ? i * p.hw : 0u;
        const unsigned limit = p.per_image ? p.hw : p.m;
        const unsigned end = base + (p.seg < limit - min(first, limit) ? first + p.seg : limit);
        for (unsigned m0 = base + first + (threadIdx.x >> 6) * PW; m0 < end; m0 += 4u * PW) {
            const bool mine = m0 + at.pix < end;
            unsigned img, pix;
            split_pixel(p, mine ? m0 + at.pix : end - 1, img, pix);
            float s[NG][8], v[NG][8], d[NG][8], ds[NG][8];
#pragma unroll
            for (int j = 0; j < NG; ++j) get8<XT>(p.x, img, pix, g[j], s[j]);
            if (p.y.ptr) {
#pragma unroll
                for (int j = 0; j < NG; ++j) get8<DT>(p.y, img, pix, g[j], v[j]);
            }
            if (p.d_out.ptr) {
#pragma unroll
                for (int j = 0; j < NG; ++j) get8<DT>(p.d_out, img, pix, g[j], d[j]);
            }
            if (p.d_sum.ptr) {
#pragma unroll
                for (int j = 0; j < NG; ++j) get8<XT>(p.d_sum, img, pix, g[j], ds[j]);
            } else {
#pragma unroll
                for (int j = 0; j < NG; ++j)
#pragma unroll
                    for (int e = 0; e < 8; ++e) ds[j][e] = 0.f;
            }
            if (!live) {
#pragma unroll
                for (int e = 0; e < 8; ++e) s[NG - 1][e] = v[NG - 1][e] = d[NG - 1][e] = ds[NG - 1][e] = 0.f;
            }
            float ry = 0.f;
            if (p.y.ptr) {
                if (p.post_w) ry = normalise<L, NG>(v, p, live);
#pragma unroll
                for (int j = 0; j < NG; ++j) {
                    float w[8], b[8], q[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) { w[e] = 1.f; b[e] = 0.f; q[e] = 1.f; }
                    if (p.post_w) vec8(p.post_w + g[j] * 8, w);
                    if (p.post_b) vec8(p.post_b + g[j] * 8, b);
                    if (p.gate) vec8(p.gate + (unsigned long long)img * p.gate_stride + g[j] * 8, q);
#pragma unroll
                    for (int e = 0; e < 8; ++e) s[j][e] += (p.res_scale * q[e]) * (v[j][e] * w[e] + b[e]);
                }
                if (!live) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) s[NG - 1][e] = 0.f;
                }
            }
            if (p.d_out.ptr) {
                const float rs = normalise<L, NG>(s, p, live);
                float dot = 0.f, tot = 0.f;
#pragma unroll
                for (int j = 0; j < NG; ++j) {
                    float w[8];
                    vec8(p.pre_w + g[j] * 8, w);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        if (mine) {
                            sums[kPreW][j][e] += d[j][e] * s[j][e];
                            sums[kPreB][j][e] += d[j][e];
                        }
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
            if (p.dx.ptr && mine) {
#pragma unroll
                for (int j = 0; j < NG; ++j)
                    if (j < NG - 1 || live) put8<XT>(p.dx, img, pix, g[j], ds[j]);
            }
            if (p.y.ptr) {
                float dot = 0.f, tot = 0.f;
#pragma unroll
                for (int j = 0; j < NG; ++j) {
                    float w[8], b[8], q[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) { w[e] = 1.f; b[e] = 0.f; q[e] = 1.f; }
                    if (p.post_w) vec8(p.post_w + g[j] * 8, w);
                    if (p.post_b) vec8(p.post_b + g[j] * 8, b);
                    if (p.gate) vec8(p.gate + (unsigned long long)img * p.gate_stride + g[j] * 8, q);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float dv = (p.res_scale * q[e]) * ds[j][e];
                        if (mine) {
                            gsum[j][e] += ds[j][e] * (v[j][e] * w[e] + b[e]);
                            sums[kPostW][j][e] += dv * v[j][e];
                            sums[kPostB][j][e] += dv;
                        }
                        d[j][e] = j < NG - 1 || live ? dv * w[e] : 0.f;
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
                        for (int e = 0; e < 8; ++e) d[j][e] = ry * (d[j][e] - dot * v[j][e] - tot);
                }
                if (p.dy.ptr && mine) {
#pragma unroll
                    for (int j = 0; j < NG; ++j)
                        if (j < NG - 1 || live) put8<DT>(p.dy, img, pix, g[j], d[j]);
                }
            }
        }
        if (p.per_image && p.gate_part) {
            const unsigned slot = p.chunks > 1 ? blockIdx.x : i;
            join_sums<L, NG>(gsum, at, p, live, red, p.gate_part + (unsigned long long)slot * p.c);
#pragma unroll
            for (int j = 0; j < NG; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) gsum[j][e] = 0.f;
        }
    }
    float* row = p.part + (unsigned long long)blockIdx.x * p.kinds * p.c;
    int k = 0;
    if (p.post_w) join_sums<L, NG>(sums[kPostW], at, p, live, red, row + p.c * k++);
    if (p.post_b) join_sums<L, NG>(sums[kPostB], at, p, live, red, row + p.c * k++);
    if (p.d_out.ptr) join_sums<L, NG>(sums[kPreW], at, p, live, red, row + p.c * k++);
    if (p.d_out.ptr && p.pre_b) join_sums<L, NG>(sums[kPreB], at, p, live, red, row + p.c * k++);
    if (p.gate && !p.per_image) join_sums<L, NG>(gsum, at, p, live, red, row + p.c * k++);
#endif
}

// ---- host --------------------------------------------------------------------------------------------------------------
constexpr int kNormMaxC = 1024;

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
    const size_t lds = (size_t)4 * p.c * sizeof(float);
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
constexpr unsigned kNormWorkgroups = 1024;
static NormSplit norm_split(int n, long long hw, int c, bool per_image) {
    NormSplit s = {};
    norm_shape(c / 8, 2, &s.lanes, &s.ng);
    const unsigned step = 4u * (64u / (unsigned)s.lanes);  // pixels of a workgroup's iteration
    const unsigned long long span = per_image ? (unsigned long long)hw : (unsigned long long)n * hw;
    const unsigned want = per_image ? ((unsigned)n >= kNormWorkgroups ? 1u : kNormWorkgroups / (unsigned)n) : kNormWorkgroups;
    unsigned long long seg = (span + want - 1) / want;
    seg = (seg + step - 1) / step * step;
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
    const unsigned cols = (unsigned)(p.c + 31) / 32;
    if (p.kinds) {
        SumRows r = {};
        r.part = p.part; r.outer_stride = p.c; r.row_stride = (long long)p.kinds * p.c; r.rows = sp.grid; r.c = p.c;
        auto add = [&](float* dst, float scale) { if (dst) { r.dst[r.n_dst] = dst; r.scale[r.n_dst++] = scale; } };
        add(d->d_post_weight, 1.f); add(d->d_post_bias, 1.f); add(d->d_pre_weight, 1.f); add(d->d_pre_bias, 1.f);
        if (!per_image) add(d->d_gate, d->res_scale);
        hipLaunchKernelGGL(sum_rows_kernel, dim3(cols, (unsigned)p.kinds), dim3(1024), 0, s, r);
        SRMI_HIP(hipGetLastError());
    }
    if (per_image) {
        for (unsigned i = 0; i < p.n; i += 65535u) {
            SumRows r = {};
            r.part = p.gate_part + (size_t)i * sp.chunks * p.c;
            r.outer_stride = (long long)sp.chunks * p.c; r.row_stride = p.c; r.rows = sp.chunks; r.c = p.c;
            r.dst[0] = d->d_gate + (size_t)i * p.c; r.scale[0] = d->res_scale;
            hipLaunchKernelGGL(sum_rows_kernel, dim3(cols, p.n - i < 65535u ? p.n - i : 65535u), dim3(1024), 0, s, r);
            SRMI_HIP(hipGetLastError());
        }
    }
    return 0;
}
