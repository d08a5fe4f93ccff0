// The seam with norms of queries and keys and the forms of rotary positions that models have beside the
// half split over a whole head (kernel.py:209-249 of the reference, whose QK-norm is ops/norm.py): for one
// token and head
//     x      the projection, plus the bias in fp32
//     q, k   x / sqrt(mean(x^2) + eps) * w (where the model has norms), q times the attention scale
//     q, k   channel pairs of the first rotary_dim channels turned by the position's angles: (j, j +
//            rotary_dim / 2), or (2 j, 2 j + 1) interleaved; the channels behind them as they are
//     then   round to Q8.16, half to even, clamped to 24 bits
// in float64 (sums, norms and angles' products), the steps of seam_pair in its order where there is no
// norm. With cast_after_rope = 0 the cast comes before the rotation, which is then in integers.
//
// What bounds it: memory, 8 bytes a channel (205 MB for 4,096 tokens of 48 heads of 128). So a lane takes
// 8 channels of one head, two groups of 4 consecutive ones that pair up (16-byte loads and stores), a
// head of 64 takes 8 lanes, and a sum over a head is 3 or 4 DPP steps. Heads and tokens are numbered
// through, so that no lane idles whatever the head count. 4,096 tokens of 48 heads of 128 with norms: 43.5 us,
// 4.7 TB/s, the rate of a large copy; 777 tokens of 64, half interleaved, 8.4 us; one token 4.3, a launch. Rows
// that are not 16-byte aligned, or a rotary_dim that is no multiple of 8, take single words: 80 us and 12 us.
#pragma once

#include "insitu_internal.h"
#include "wave.h"

namespace insitu {

struct SeamHeads {
    const float *p, *bias, *w_q, *w_k;
    int32_t n_q, n_kv, d, rotary;
    const int64_t *pos;
    int64_t pos0;
    const int64_t *cos_t, *sin_t;
    int64_t max_pos;
    int32_t frac, interleaved, cast_after_rope;
    uint32_t units;                       // tokens times heads
    double inv_heads, attn_scale, eps;
    int32_t *q, *k, *v;
    unsigned long long *sat, *range_err;
};

// Sum over the LPH lanes (a power of two up to 64) of a head, in each of them.
template <int LPH>
__device__ __forceinline__ double head_sum(double v) {
    auto dpp = [&](auto ctrl) {
        return __longlong_as_double(dpp64<decltype(ctrl)::value>(0, __double_as_longlong(v)));
    };
    if constexpr (LPH >= 2) v += dpp(std::integral_constant<int, DPP_QUAD_1032>{});
    if constexpr (LPH >= 4) v += dpp(std::integral_constant<int, DPP_QUAD_2301>{});
    if constexpr (LPH >= 8) v += dpp(std::integral_constant<int, DPP_ROW_HALF_MIRROR>{});
    if constexpr (LPH >= 16) v += dpp(std::integral_constant<int, DPP_ROW_MIRROR>{});
    if constexpr (LPH >= 32) v += __shfl_xor(v, 16);
    if constexpr (LPH >= 64) v += __shfl_xor(v, 32);
    return v;
}

__device__ __forceinline__ int32_t seam_fixed(double a, uint32_t &sat) {
#pragma clang fp contract(off)
    const double r = rint(a * 65536.0);
    const double lo = -(double)(1 << 23), hi = (double)((1 << 23) - 1);
    sat += r < lo || r > hi ? 1u : 0u;
    return (int32_t)(r < lo ? lo : r > hi ? hi : r);
}

// VEC channel pairs a lane, LPH lanes a head: d = 2 VEC LPH. VEC = 4 where rows are 16-byte aligned and
// rotary_dim is a multiple of 8 (a lane's four pairs then rotate all or not at all).
template <int VEC, int LPH>
__global__ void __launch_bounds__(256) seam_heads_kernel(SeamHeads a) {
#pragma clang fp contract(off)
    constexpr int ITER = VEC == 4 ? 2 : 4, HEADS = 256 / LPH;
    const int l = threadIdx.x % LPH, j0 = VEC * l, d = a.d, half = a.rotary / 2, heads = a.n_q + 2 * a.n_kv;
    const bool turn = j0 < half, il = turn && a.interleaved != 0;
    // the first channels of the two groups; interleaved they are 2 VEC consecutive ones
    const int ca = !turn ? a.rotary + j0 - half : il ? 2 * j0 : j0;
    const int cb = !turn ? ca + (d - a.rotary) / 2 : il ? ca + VEC : ca + half;
    uint32_t sat = 0;
    float x[ITER][2][VEC];
    uint32_t un[ITER];
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        un[i] = blockIdx.x * (uint32_t)(HEADS * ITER) + i * HEADS + threadIdx.x / LPH;
        if (un[i] >= a.units) continue;
        const float *row = a.p + (int64_t)un[i] * d;
        if constexpr (VEC == 4) {
            *(float4 *)x[i][0] = *(const float4 *)(row + ca);
            *(float4 *)x[i][1] = *(const float4 *)(row + cb);
        } else {
            x[i][0][0] = row[ca];
            x[i][1][0] = row[cb];
        }
    }
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        const bool in = un[i] < a.units;
        const uint32_t u = in ? un[i] : a.units - 1;
        int64_t t = (int64_t)((double)u * a.inv_heads);       // within one of u / heads
        int h = (int)((int64_t)u - t * heads);
        if (h < 0) {
            h += heads;
            --t;
        } else if (h >= heads) {
            h -= heads;
            ++t;
        }
        const int kind = h < a.n_q ? 0 : h < a.n_q + a.n_kv ? 1 : 2;
        if (a.bias && in) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                x[i][0][e] = x[i][0][e] + a.bias[h * d + ca + e];
                x[i][1][e] = x[i][1][e] + a.bias[h * d + cb + e];
            }
        }
        double y[2][VEC];
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int e = 0; e < VEC; ++e) y[k][e] = in ? (double)x[i][k][e] : 0.0;
        const float *w = kind == 0 ? a.w_q : kind == 1 ? a.w_k : nullptr;
        if (a.w_q || a.w_k) {                                  // (uniform: the sum takes every lane)
            double ss = 0.0;
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int e = 0; e < VEC; ++e) ss += y[k][e] * y[k][e];
            ss = head_sum<LPH>(ss);
            if (w) {
                const double inv = 1.0 / sqrt(ss / d + a.eps);
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    y[0][e] = y[0][e] * inv * (double)w[ca + e];
                    y[1][e] = y[1][e] * inv * (double)w[cb + e];
                }
            }
        }
        if (kind == 0) {
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int e = 0; e < VEC; ++e) y[k][e] = y[k][e] * a.attn_scale;
        }
        if (!in) continue;
        int32_t o[2][VEC];
        const int64_t ps = a.pos ? a.pos[t] : a.pos0 + t;
        if (kind != 2 && (ps < 0 || ps >= a.max_pos)) {
            if (l == 0) atomicAdd(a.range_err, 1ull);
            continue;
        }
        if (kind == 2 || !turn) {
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int e = 0; e < VEC; ++e) o[k][e] = seam_fixed(y[k][e], sat);
        } else {
            if (il) {
                // the groups hold pairs in turn: (first, second) of pair e in the lower's and the upper's order
                double z[2][VEC];
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    z[0][e] = y[2 * e / VEC][2 * e % VEC];
                    z[1][e] = y[(2 * e + 1) / VEC][(2 * e + 1) % VEC];
                }
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) y[k][e] = z[k][e];
            }
            int64_t c[VEC], s[VEC];
            const int64_t *cp = a.cos_t + ps * half + j0, *sp = a.sin_t + ps * half + j0;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                c[e] = cp[e];
                s[e] = sp[e];
            }
            const double unit = __longlong_as_double((int64_t)(1023 - a.frac) << 52);   // 2^-frac
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                if (a.cast_after_rope) {
                    const double cf = (double)c[e] * unit, sf = (double)s[e] * unit;
                    const double e0 = y[0][e] * cf, e1 = y[1][e] * sf, e2 = y[0][e] * sf, e3 = y[1][e] * cf;
                    o[0][e] = seam_fixed(e0 - e1, sat);
                    o[1][e] = seam_fixed(e2 + e3, sat);
                } else {
                    const int64_t lo = seam_fixed(y[0][e], sat), hi = seam_fixed(y[1][e], sat);
                    o[0][e] = (int32_t)((lo * c[e] - hi * s[e]) >> a.frac);
                    o[1][e] = (int32_t)((lo * s[e] + hi * c[e]) >> a.frac);
                }
            }
            if (il) {
                int32_t z[2][VEC];
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    z[2 * e / VEC][2 * e % VEC] = o[0][e];
                    z[(2 * e + 1) / VEC][(2 * e + 1) % VEC] = o[1][e];
                }
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) o[k][e] = z[k][e];
            }
        }
        int32_t *dst = kind == 0 ? a.q + (t * a.n_q + h) * d
                                 : kind == 1 ? a.k + (t * a.n_kv + h - a.n_q) * d : a.v + (t * a.n_kv + h - a.n_q - a.n_kv) * d;
        if constexpr (VEC == 4) {
            *(int4 *)(dst + ca) = *(const int4 *)o[0];
            *(int4 *)(dst + cb) = *(const int4 *)o[1];
        } else {
            dst[ca] = o[0][0];
            dst[cb] = o[1][0];
        }
    }
    if (sat) atomicAdd(a.sat, (unsigned long long)sat);
}

inline hipError_t launch_seam_heads(hipStream_t s, const SeamHeads &a) {
    // (16 bytes a lane of every row: of p and of what is written)
    const uintptr_t at = (uintptr_t)a.p | (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v;
    const bool vec = (at & 15) == 0 && a.rotary % 8 == 0;
    const int lph = vec ? a.d / 8 : a.d / 2, per = (256 / lph) * (vec ? 2 : 4);
    const dim3 grid((a.units + per - 1) / per), block(256);
#define INSITU_SEAM(V, L) \
    if (vec == (V == 4) && lph == L) hipLaunchKernelGGL((seam_heads_kernel<V, L>), grid, block, 0, s, a)
    INSITU_SEAM(4, 2);
    INSITU_SEAM(4, 4);
    INSITU_SEAM(4, 8);
    INSITU_SEAM(4, 16);
    INSITU_SEAM(1, 8);
    INSITU_SEAM(1, 16);
    INSITU_SEAM(1, 32);
    INSITU_SEAM(1, 64);
#undef INSITU_SEAM
    return hipGetLastError();
}

}  // namespace insitu
