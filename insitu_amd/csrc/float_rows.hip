// Floating keys and values in and out of the compressed cache: a dense cache's rows cast to Q8.16 (to_fixed,
// ops/convert.py:44-57), rotated (ops/rotate.py:170-197), encoded and packed (ops/quantize.py:164-252) behind
// each sequence; and a cache's rows as floating ones, centroid times norm turned back by the rotation's
// inverse (the decode of ops/quantize.py:214-222 and ops/rotate.py:199-231, not in fixed point but in floating).
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "row_codec.h"

namespace insitu {
namespace fr {

template <class T>
__device__ __forceinline__ float to_f32(T x) {
    return (float)x;
}
// Q8.16, half to even, at the 24 bits' ends where it lies beyond them; NaN is 0. sat: whether it did not fit
__device__ __forceinline__ int32_t to_q16(float f, bool &sat) {
    const float r = rintf(f * 65536.0f);
    sat = !(r >= -8388608.0f && r <= 8388607.0f);
    return r != r ? 0 : (int32_t)fminf(fmaxf(r, -8388608.0f), 8388607.0f);
}

constexpr int WAVES = 4;

// Any format of up to two rounds: a wave a row, lane = channel.
template <int CPL, class T>
__global__ void __launch_bounds__(64 * WAVES) append_kernel(Geom g, const Tables *__restrict__ tabs, FloatRows k, FloatRows v,
                                                            int n_tok, int seq_lo, int seq_hi, const int64_t *__restrict__ len_in,
                                                            int64_t *len_out, int64_t *len_now, int rounds, RotSigns sg,
                                                            int count, DevStats *st) {
    __shared__ uint8_t codes[WAVES][2][MAX_D];
    __shared__ int64_t bnd[2][255];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    stage_bounds(tabs, g, bnd);
    if (blockIdx.x == 0) {                             // the lengths, as an append of wire rows leaves them
        for (int i = threadIdx.x; i < g.batch; i += blockDim.x)
            len_out[i] = len_now[i] = len_in[i] + ((i >= seq_lo && i < seq_hi) ? n_tok : 0);
    }
    __syncthreads();
    const int64_t rows = (int64_t)(seq_hi - seq_lo) * n_tok * g.n_kv;
    for (int64_t r = (int64_t)blockIdx.x * WAVES + wv; r < rows; r += (int64_t)gridDim.x * WAVES) {
        const int h = (int)(r % g.n_kv);
        const int64_t tb = r / g.n_kv;
        const int t = (int)(tb % n_tok), b = (int)(tb / n_tok);
        const int64_t pos = len_in[seq_lo + b] + t;
        int64_t norm[2];
        unsigned long long lost = 0;
#pragma unroll
        for (int f = 0; f < 2; ++f) {
            const FloatRows &src = f == 0 ? k : v;
            const T *p = (const T *)src.p + b * src.seq + t * src.tok + h * src.head;
            int32_t x[CPL], y[CPL];
#pragma unroll
            for (int j = 0; j < CPL; ++j) {
                const int ch = lane + 64 * j;
                bool sat = false;
                x[j] = ch < g.d ? to_q16(to_f32(p[ch]), sat) : 0;
                lost += sat ? 1 : 0;
            }
            rotate_loaded<CPL>(x, g.d, rounds, sg, y, nullptr);
            int64_t z[CPL];
#pragma unroll
            for (int j = 0; j < CPL; ++j) z[j] = y[j];
            norm[f] = encode_field<CPL>(z, g.d, g.norm_frac, bnd[f], (1 << (f == 0 ? g.kb : g.vb)) - 1, codes[wv][f]);
        }
        if (count && lost) atomicAdd(&st->range_errors, lost);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        if (pos < g.capacity)
            pack_store_row(g, codes[wv], norm[0], norm[1], seq_lo + b, h, pos);
        else if (lane == 0)                            // the host checks capacity first; this only guards memory
            atomicAdd(&st->fault, 1ull);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
}

// Any format of up to two rounds: a wave a row, lane = channel. A field's codes may run over its planes.
template <int CPL, class T>
__global__ void __launch_bounds__(64 * WAVES) read_kernel(Geom g, const Tables *__restrict__ tabs, FloatRows k, FloatRows v,
                                                          int64_t t0, int64_t n, int seq_lo, int seq_hi,
                                                          const int64_t *__restrict__ len, int rounds, RotSigns sg) {
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t rows = (seq_hi - seq_lo) * n * g.n_kv;
    const double root = rsqrt((double)g.d);
    for (int64_t r = (int64_t)blockIdx.x * WAVES + wv; r < rows; r += (int64_t)gridDim.x * WAVES) {
        const int h = (int)(r % g.n_kv);
        const int64_t t = r / g.n_kv % n;
        const int b = (int)(r / g.n_kv / n);
        if (t0 + t >= len[seq_lo + b]) continue;
        auto byte = [&](int i) { return (uint32_t)*((const uint8_t *)row_word_ptr(g, seq_lo + b, h, t0 + t, i / 4) + i % 4); };
#pragma unroll
        for (int f = 0; f < 2; ++f) {
            const FloatRows &dst = f == 0 ? k : v;
            const int bits = f == 0 ? g.kb : g.vb, field = f == 0 ? 0 : g.key_bytes;
            const int at = g.key_bytes + g.value_bytes + 2 * f;
            const int64_t norm = sext16(byte(at) | byte(at + 1) << 8);
            double x[CPL];
#pragma unroll
            for (int j = 0; j < CPL; ++j) {
                const int ch = lane + 64 * j;
                x[j] = 0.0;
                if (ch >= g.d) continue;
                const int o = ch * bits;
                uint32_t c = byte(field + (o >> 3));
                if ((o & 7) + bits > 8) c |= byte(field + (o >> 3) + 1) << 8;
                x[j] = (double)(f == 0 ? tabs->kc : tabs->vc)[(c >> (o & 7)) & ((1u << bits) - 1)];
            }
            for (int i = rounds - 1; i >= 0; --i) {
                for (int o = 1; o < g.d && o < 64; o <<= 1) {
#pragma unroll
                    for (int j = 0; j < CPL; ++j) {
                        const double y = __shfl_xor(x[j], o);
                        x[j] = lane & o ? y - x[j] : x[j] + y;
                    }
                }
                if (CPL == 2 && g.d == 128) {
                    const double a = x[0], c = x[CPL - 1];
                    x[0] = a + c;
                    x[CPL - 1] = a - c;
                }
#pragma unroll
                for (int j = 0; j < CPL; ++j) {
                    const int ch = lane + 64 * j;
                    const uint64_t w = ch < 64 ? (i == 0 ? sg.s0a : sg.s1a) : (i == 0 ? sg.s0b : sg.s1b);
                    x[j] *= (w >> (ch & 63)) & 1 ? -root : root;
                }
            }
            T *p = (T *)dst.p + b * dst.seq + t * dst.tok + h * dst.head;
#pragma unroll
            for (int j = 0; j < CPL; ++j) {
                const int ch = lane + 64 * j;
                if (ch < g.d) p[ch] = (T)(float)(x[j] * (double)norm * 0x1p-24);
            }
        }
    }
}

template <class F>
hipError_t by_type(int type, F &&f) {
    switch (type) {
        case INSITU_F32: f(float{}); break;
        case INSITU_F16: f(__half{}); break;
        case INSITU_BF16: f(__hip_bfloat16{}); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

unsigned grid_of(int64_t rows) {
    const int64_t blocks = (rows + WAVES - 1) / WAVES;
    return (unsigned)(blocks < 4096 ? blocks : 4096);
}

}  // namespace fr

hipError_t launch_append_float(hipStream_t s, const Geom &g, const Tables *t, const FloatRows &k, const FloatRows &v, int type,
                               int n_tok, int seq_lo, int seq_hi, const int64_t *len_in, int64_t *len_out, int64_t *len_now,
                               int rounds, const uint64_t (*signs)[2], bool count, DevStats *st) {
    const int64_t rows = (int64_t)(seq_hi - seq_lo) * n_tok * g.n_kv;
    if (rows <= 0) return hipSuccess;
    if (rounds < 0 || rounds > 2) return hipErrorInvalidValue;
    const RotSigns sg = rounds ? rot_signs(rounds, signs) : RotSigns{};
    return fr::by_type(type, [&](auto x) {
        using T = decltype(x);
        if (g.d <= 64)
            hipLaunchKernelGGL((fr::append_kernel<1, T>), dim3(fr::grid_of(rows)), dim3(64 * fr::WAVES), 0, s, g, t, k, v, n_tok,
                               seq_lo, seq_hi, len_in, len_out, len_now, rounds, sg, count ? 1 : 0, st);
        else
            hipLaunchKernelGGL((fr::append_kernel<2, T>), dim3(fr::grid_of(rows)), dim3(64 * fr::WAVES), 0, s, g, t, k, v, n_tok,
                               seq_lo, seq_hi, len_in, len_out, len_now, rounds, sg, count ? 1 : 0, st);
    });
}

hipError_t launch_read_float(hipStream_t s, const Geom &g, const Tables *t, const FloatRows &k, const FloatRows &v, int type,
                             int64_t t0, int64_t n, int seq_lo, int seq_hi, const int64_t *len, int rounds,
                             const uint64_t (*signs)[2]) {
    const int64_t rows = (seq_hi - seq_lo) * n * g.n_kv;
    if (rows <= 0) return hipSuccess;
    if (rounds < 0 || rounds > 2) return hipErrorInvalidValue;
    const RotSigns sg = rounds ? rot_signs(rounds, signs) : RotSigns{};
    return fr::by_type(type, [&](auto x) {
        using T = decltype(x);
        if (g.d <= 64)
            hipLaunchKernelGGL((fr::read_kernel<1, T>), dim3(fr::grid_of(rows)), dim3(64 * fr::WAVES), 0, s, g, t, k, v, t0, n,
                               seq_lo, seq_hi, len, rounds, sg);
        else
            hipLaunchKernelGGL((fr::read_kernel<2, T>), dim3(fr::grid_of(rows)), dim3(64 * fr::WAVES), 0, s, g, t, k, v, t0, n,
                               seq_lo, seq_hi, len, rounds, sg);
    });
}

}  // namespace insitu
