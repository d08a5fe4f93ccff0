// Floating keys and values in and out of the compressed cache: a dense cache's rows cast to Q8.16 (to_fixed,
// ops/convert.py:44-57), rotated (ops/rotate.py:170-197), encoded and packed (ops/quantize.py:164-252) behind
// each sequence; and a cache's rows as floating ones, centroid times norm turned back by the rotation's
// inverse (the decode of ops/quantize.py:214-222 and ops/rotate.py:199-231, not in fixed point but in floating).
//
// The rotation is a product with +-1 and so one of signed bytes on the matrix cores, exactly: a Q8.16 value and a
// centroid are three balanced digits, 16 rows a wave and product, and the outputs' order is chosen so that a lane
// holds D / 4 channels of a row side by side. What it loads, packs or stores are then whole words, with no
// exchange through LDS.
//
// What bounds it. Reading: memory, 32,767 tokens of 8 heads of 64 into bfloat16 19.0 us, 4.25 TB/s where a copy has 4.68
// (a wave a row and its butterfly in floating point 292 us). Writing: VALU issue, 76 % of the SIMDs' cycles in 40 of
// 41.9 us for the same rows (405 a wave a row), 1,200 instructions a tile of 16 rows: the cast and its digits, the
// exact norm, the codes by a bisection of the boundaries and their packing. Comparisons in place of signs 49 us; the boundaries' selects as v_bfi by hand 49; a norm in 32 bits with the exact one where it is close 40.5, not
// worth a second way. Small calls are the host's: 65 tokens 6.6 us of kernel in 16, 100 read 4.5 in 13.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <cstdlib>
#include <type_traits>

#include "digits.h"
#include "row_codec.h"

namespace insitu {
namespace fr {

template <class T>
__device__ __forceinline__ float to_f32(T x) {
    return (float)x;
}
// Q8.16, half to even, at the 24 bits' ends where it lies beyond them; NaN is 0 (as the conversion to 32 bits gives
// it, which takes their ends beyond them).
__device__ __forceinline__ int32_t to_q16(float f) {
    const float r = rintf(f * 65536.0f);
    int32_t x;
    asm("v_cvt_i32_f32 %0, %1" : "=v"(x) : "v"(r));
    return x < -(1 << 23) ? -(1 << 23) : x > (1 << 23) - 1 ? (1 << 23) - 1 : x;
}
// Whether it did not fit.
__device__ __forceinline__ bool lost_q16(float f) {
    const float r = rintf(f * 65536.0f);
    return !(r >= -8388608.0f && r <= 8388607.0f);
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
                const float y = ch < g.d ? to_f32(p[ch]) : 0.0f;
                x[j] = to_q16(y);
                lost += lost_q16(y) ? 1 : 0;
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

// 1 / 2^24 (Q15 times Q9) and 1 / sqrt d a round. A value is a whole number times the norm and this, the same
// roundings in either kernel: the number's, the scale's two and the product's.
// (rounded to 32 bits before it is to 16: the compiler may not join the two.)
__host__ __device__ constexpr float unit_of(int d, int rounds) {
    return (float)(0x1p-24 / (rounds == 2 ? d : rounds == 1 ? (d == 64 ? 8.0 : 11.313708498984761) : 1.0));
}

__device__ __forceinline__ float product(float a, float b) {
#pragma clang fp contract(off)
    float y = a * b;
    asm("" : "+v"(y));
    return y;
}

// Any format of up to two rounds: a wave a row, lane = channel. A field's codes may run over its planes.
template <int CPL, class T>
__global__ void __launch_bounds__(64 * WAVES) read_kernel(Geom g, const Tables *__restrict__ tabs, FloatRows k, FloatRows v,
                                                          int64_t t0, int64_t n, int seq_lo, int seq_hi,
                                                          const int64_t *__restrict__ len, int rounds, RotSigns sg) {
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t rows = (seq_hi - seq_lo) * n * g.n_kv;
    const float unit = unit_of(g.d, rounds);
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
                for (int o = 1; o < 64; o <<= 1) {
#pragma unroll
                    for (int j = 0; j < CPL; ++j) {
                        const double y = __shfl_xor(x[j], o);
                        x[j] = lane & o ? y - x[j] : x[j] + y;
                    }
                }
                if (CPL == 2) {
                    const double a = x[0], c = x[CPL - 1];
                    x[0] = a + c;
                    x[CPL - 1] = a - c;
                }
#pragma unroll
                for (int j = 0; j < CPL; ++j) {
                    const int ch = lane + 64 * j;
                    const uint64_t w = ch < 64 ? (i == 0 ? sg.s0a : sg.s1a) : (i == 0 ? sg.s0b : sg.s1b);
                    x[j] = (w >> (ch & 63)) & 1 ? -x[j] : x[j];
                }
            }
            T *p = (T *)dst.p + b * dst.seq + t * dst.tok + h * dst.head;
#pragma unroll
            for (int j = 0; j < CPL; ++j) {
                const int ch = lane + 64 * j;
                if (ch < g.d) p[ch] = (T)product((float)x[j], (float)norm * unit);      // (x: whole, below 2^34)
            }
        }
    }
}

// -- 16 rows a wave: one round, keys of 2 to 4 bits, values of 1 to 3 -----------------------------------------

// What every tile of 16 tokens has in common.
struct Tiles {
    Geom g;
    FloatRows k, v;
    const int64_t *len_in;
    int64_t *len_out, *len_now;                        // (append: null otherwise)
    int64_t t0, n;                                     // rows of a sequence
    uint32_t tiles;                                    // of all
    int32_t per;                                       // of a (sequence, KV head)
    int32_t seq_lo, seq_hi, type, count;               // count: values that do not fit
    uint64_t sa, sb;                                   // the rotation's signs of channels 0 .. 63 and 64 .. 127
    double bnd[2][15];                                 // boundaries / 2^8 (append)
    DevStats *st;
};

// The channel that output m = 4 a + i of product c is, lane group a of the result holding it. SIDE: D / 4 channels side by
// side a lane, for codes to be packed; otherwise a row's four lanes side by side, 16 bytes each, for stores: 4 channels of
// 32 bits (LANES4) or, of two products, 8 of 16 (LANES8).
enum Order { SIDE, LANES4, LANES8 };
__device__ __forceinline__ int channel(Order how, int D, int c, int a, int i) {
    return how == SIDE ? D / 4 * a + 4 * c + i : how == LANES4 ? 16 * c + 4 * a + i : 32 * (c / 2) + 8 * a + 4 * (c % 2) + i;
}
// The products' left operand: lane = (output m, 16 inputs from D / 4 grp + 16 b on), +-1 bytes. Of input j and
// output o the sign is the parity of o & j times that of the rotation's diagonal, at the input (forward) or at the
// output (inverse). IDENTITY: 1 where they are the same.
enum Turn { FORWARD, INVERSE, IDENTITY };
template <int D>
__device__ __forceinline__ void turn_row(Turn how, Order order, uint64_t sa, uint64_t sb, int c, v4i (&A)[D / 64]) {
    const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
    const uint32_t o = (uint32_t)channel(order, D, c, col >> 2, col & 3);
    // bit j: the parity of o & j, j < 16
    const uint32_t w = ((o & 1) ? 0xAAAAu : 0u) ^ ((o & 2) ? 0xCCCCu : 0u) ^ ((o & 4) ? 0xF0F0u : 0u) ^ ((o & 8) ? 0xFF00u : 0u);
    const uint32_t so = (uint32_t)((o < 64 ? sa : sb) >> (o & 63)) & 1u;
#pragma unroll
    for (int b = 0; b < D / 64; ++b) {
        const uint32_t j0 = (uint32_t)(D / 4 * grp + 16 * b);
        const uint32_t hi = (uint32_t)__popc((o >> 4) & (j0 >> 4)) & 1u;
        uint32_t x = w ^ (hi ? 0xFFFFu : 0u);
        x ^= how == FORWARD ? (uint32_t)((j0 < 64 ? sa : sb) >> (j0 & 63)) & 0xFFFFu : so ? 0xFFFFu : 0u;
        const uint32_t same = o >> 4 == j0 >> 4 ? 1u << (o & 15) : 0u;
        if (how == IDENTITY) x = same;
#pragma unroll
        for (int d = 0; d < 4; ++d) {                  // four bits to four bytes
            const uint32_t y = ((x >> (4 * d) & 15u) * 0x00204081u) & 0x01010101u;
            A[b][d] = (int)(how == IDENTITY ? y : 0x01010101u + 0xFEu * y);        // 0: 1, 1: -1
        }
    }
}
// All of them into LDS, a wave the c's of its number; the caller synchronises.
template <int D>
__device__ __forceinline__ void turn_rows(Turn how, Order order, uint64_t sa, uint64_t sb, v4i (*A)[D / 64][64]) {
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
    for (int c = 0; c < D / 16; c += WAVES) {
        v4i a[D / 64];
        turn_row<D>(how, order, sa, sb, c + wv, a);
#pragma unroll
        for (int b = 0; b < D / 64; ++b) A[c + wv][b][lane] = a[b];
    }
}

// What a tile's rows are: 16 tokens of a (sequence, KV head).
struct Tile {
    int b, h, t;                                       // sequence of the call; KV head; the lane's row, of n
    bool there;                                        // (a lane past the end holds the last row again)
    __device__ __forceinline__ Tile(const Tiles &J, uint32_t i) {
        const uint32_t chain = i / (uint32_t)J.per, first = (i - chain * (uint32_t)J.per) * 16;
        b = (int)(chain / (uint32_t)J.g.n_kv);
        h = (int)(chain - (uint32_t)b * (uint32_t)J.g.n_kv);
        t = (int)first + (int)(threadIdx.x & 15);
        there = t < J.n;
        t = there ? t : (int)J.n - 1;
    }
    __device__ __forceinline__ int64_t at(const FloatRows &r) const { return b * r.seq + t * r.tok + h * r.head; }
};

// A lane's floating values: D / 4 channels from D / 4 grp on.
template <int D>
struct Floats {
    uint4 w[D / 16];                                   // (16-bit types: the first half)
    __device__ __forceinline__ void load(const void *p, int64_t at, int type) {
        const int grp = (threadIdx.x & 63) >> 4;
        if (type == INSITU_F32) {
#pragma unroll
            for (int b = 0; b < D / 64; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) w[4 * b + i] = *(const uint4 *)((const float *)p + at + D / 4 * grp + 16 * b + 4 * i);
        } else {
#pragma unroll
            for (int b = 0; b < D / 64; ++b)
#pragma unroll
                for (int i = 0; i < 2; ++i) w[2 * b + i] = *(const uint4 *)((const uint16_t *)p + at + D / 4 * grp + 16 * b + 8 * i);
        }
    }
    // the 16 of block b
    __device__ __forceinline__ void get(int b, int type, float (&x)[16]) const {
        if (type == INSITU_F32) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[4 * i] = __uint_as_float(w[4 * b + i].x), x[4 * i + 1] = __uint_as_float(w[4 * b + i].y);
                x[4 * i + 2] = __uint_as_float(w[4 * b + i].z), x[4 * i + 3] = __uint_as_float(w[4 * b + i].w);
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t y[4] = {w[2 * b + i].x, w[2 * b + i].y, w[2 * b + i].z, w[2 * b + i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (type == INSITU_BF16) {
                    x[8 * i + 2 * j] = __uint_as_float(y[j] << 16);
                    x[8 * i + 2 * j + 1] = __uint_as_float(y[j] & 0xFFFF0000u);
                } else {
                    x[8 * i + 2 * j] = (float)__builtin_bit_cast(_Float16, (uint16_t)y[j]);
                    x[8 * i + 2 * j + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(y[j] >> 16));
                }
            }
        }
    }
};

// N bits from bit N grp of a row's field (planes from `plane` on) of the lane's row: w holds them.
template <int N>
__device__ __forceinline__ void store_bits(const Geom &g, uint8_t *head, int plane, int field_bytes, int64_t pos, bool there,
                                           const uint32_t (&w)[(N + 31) / 32]) {
    const int lane = threadIdx.x & 63, grp = lane >> 4;
    auto word = [&](int i) {                           // dword i of the field
        const int p = i >> 2, width = field_bytes - 16 * p < 16 ? field_bytes - 16 * p : 16;
        return (uint32_t *)(head + (plane + p) * g.span + pos * width + 4 * (i & 3));
    };
    if constexpr (N == 128 || N == 64) {               // (whole, and on their size's boundary)
        if constexpr (N == 128) {
            if (there) *(uint4 *)word(4 * grp) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
            if (there) *(uint2 *)word(2 * grp) = make_uint2(w[0], w[1]);
        }
    } else if constexpr (N % 32 == 0) {
#pragma unroll
        for (int i = 0; i < N / 32; ++i)
            if (there) *word(N / 32 * grp + i) = w[i];
    } else {                                           // two lanes' make whole words
        const uint32_t low = (uint32_t)__shfl_xor((int)w[0], 16);
        if constexpr (N == 16) {
            if (there && !(grp & 1)) *word(grp >> 1) = (w[0] & 0xFFFFu) | low << 16;
        } else {
            static_assert(N == 48, "a lane's codes");
            const int i = 3 * (grp >> 1);
            if (there && !(grp & 1)) {
                *word(i) = w[0];
                *word(i + 1) = (w[1] & 0xFFFFu) | low << 16;
            }
            if (there && (grp & 1)) *word(i + 2) = w[0] >> 16 | w[1] << 16;
        }
    }
}

// One field of a tile's rows: rotated, its norm, its codes of BITS bits. Returns the norm.
template <int D, int BITS>
__device__ __forceinline__ int32_t append_field(const Tiles &J, const double *bnd, const Floats<D> &f, const v4i (*A)[D / 64][64],
                                                uint32_t &lost, uint32_t (&w)[(D / 4 * BITS + 31) / 32]) {
    // digits 0 to 2, and digit 3 of the few values above 0x7F7F7F, of which it is 1
    v4i xd[4][D / 64];
    uint32_t any3 = 0;
#pragma unroll
    for (int b = 0; b < D / 64; ++b) {
        float x[16];
        uint32_t z[16];
        if (J.type == INSITU_F32)
            f.get(b, INSITU_F32, x);
        else if (J.type == INSITU_BF16)
            f.get(b, INSITU_BF16, x);
        else
            f.get(b, INSITU_F16, x);
#pragma unroll
        for (int i = 0; i < 16; ++i) z[i] = balanced(to_q16(x[i]));
        if (J.count) {
#pragma unroll
            for (int i = 0; i < 16; ++i) lost += lost_q16(x[i]) ? 1 : 0;
        }
#pragma unroll
        for (int d = 0; d < 4; ++d) {                  // four words' bytes to three digits' words
            const uint32_t *y = z + 4 * d;
            const uint32_t e = perm(y[1], y[0], 0x05010400u), h = perm(y[3], y[2], 0x05010400u);
            xd[0][b][d] = (int)perm(h, e, 0x05040100u);
            xd[1][b][d] = (int)perm(h, e, 0x07060302u);
            const uint32_t i = perm(y[1], y[0], 0x07030602u), j = perm(y[3], y[2], 0x07030602u);
            xd[2][b][d] = (int)perm(j, i, 0x05040100u);
            xd[3][b][d] = (int)perm(j, i, 0x07060302u);
            any3 |= (uint32_t)xd[3][b][d];
        }
    }
    const bool four = __ballot(any3 != 0) != 0;
    int ln = threadIdx.x & 63;                         // (opaque, so that A is read where it is used)
    asm volatile("" : "+v"(ln));
    int32_t y[D / 4];                                  // the lane's channels: at most 2^30 before the scale, 2^27 behind it
    int64_t sq = 0;
    auto turn = [&](auto wide) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
            v4i T = {0, 0, 0, 0};
#pragma unroll
            for (int l = decltype(wide)::value ? 3 : 2; l >= 0; --l) {
                if (l < (decltype(wide)::value ? 3 : 2)) T = T << 8;
#pragma unroll
                for (int b = 0; b < D / 64; ++b) T = mma(A[c][b][ln], xd[l][b], T);
            }
            // 1 / sqrt d, floored: a shift, or (v 2896) >> 15
#pragma unroll
            for (int i = 0; i < 4; ++i) y[4 * c + i] = D == 64 ? T[i] >> 3 : __mulhi(T[i], 2896 << 17);
        }
    };
    if (four)
        turn(std::true_type{});
    else
        turn(std::false_type{});
#pragma unroll
    for (int i = 0; i < D / 4; ++i) sq += (int64_t)y[i] * y[i];
    sq += xor_lane64<16>(sq, threadIdx.x & 63);
    sq += xor_lane64<32>(sq, threadIdx.x & 63);
    int64_t n64 = rshift_even(isqrt64(sq >> (D == 64 ? 6 : 7)), QK_FRAC - 9);
    const int32_t norm = n64 > 32767 ? 32767 : (int32_t)n64;
    // y 2^8 > norm b is y > floor(norm b / 2^8), below 2^30 as the boundaries are below 2^23
    constexpr int NB = (1 << BITS) - 1;
    int32_t t[NB];
    const double nd = (double)norm;
#pragma unroll
    for (int i = 0; i < NB; ++i) t[i] = (int32_t)floor(nd * bnd[i]);
    // the codes by bisection (the boundaries do not decrease) on the signs of t - y, which do not overflow: a sign goes
    // into the word by one instruction (the last code's lowest bit comes last), chooses by another two, and comparisons,
    // whose results are scalars, would have to be waited for
    int left = D / 4 * BITS;                           // bits to come
    uint32_t x = 0;
    auto push = [&](int32_t d) __attribute__((always_inline)) {
        x = __builtin_amdgcn_alignbit(x, (uint32_t)d, 31);
        if (--left % 32 == 0) w[left / 32] = x;
    };
    auto pick = [](int32_t d, int32_t a, int32_t b) __attribute__((always_inline)) {       // a where d is negative
        const int32_t m = d >> 31;
        return (m & a) | (~m & b);
    };
#pragma unroll
    for (int i = D / 4 - 1; i >= 0; --i) {
        if constexpr (BITS == 4) {
            const int32_t d3 = t[7] - y[i];
            const int32_t d2 = pick(d3, t[11], t[3]) - y[i];
            const int32_t d1 = pick(d2, pick(d3, t[13], t[5]), pick(d3, t[9], t[1])) - y[i];
            const int32_t pr = pick(d2, pick(d3, t[12], t[4]), pick(d3, t[8], t[0]));
            const int32_t qs = pick(d2, pick(d3, t[14], t[6]), pick(d3, t[10], t[2]));
            push(d3);
            push(d2);
            push(d1);
            push(pick(d1, qs, pr) - y[i]);
        } else if constexpr (BITS == 3) {
            const int32_t d2 = t[3] - y[i];
            const int32_t d1 = pick(d2, t[5], t[1]) - y[i];
            push(d2);
            push(d1);
            push(pick(d1, pick(d2, t[6], t[2]), pick(d2, t[4], t[0])) - y[i]);
        } else if constexpr (BITS == 2) {
            const int32_t d1 = t[1] - y[i];
            push(d1);
            push(pick(d1, t[2], t[0]) - y[i]);
        } else {
            push(t[0] - y[i]);
        }
    }
    return norm;
}

template <int D, int KB, int VB>
__global__ void __launch_bounds__(64 * WAVES, D == 64 ? 4 : 2) append_tiles_kernel(Tiles J) {
    const Geom &g = J.g;
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (blockIdx.x == 0) {                             // the lengths, as an append of wire rows leaves them
        for (int i = threadIdx.x; i < g.batch; i += blockDim.x)
            J.len_out[i] = J.len_now[i] = J.len_in[i] + ((i >= J.seq_lo && i < J.seq_hi) ? J.n : 0);
    }
    // the left operands in LDS: 16 registers at d = 64, but 64 at 128
    __shared__ v4i A[D / 16][D / 64][64];
    uint32_t i = blockIdx.x * WAVES + (uint32_t)wv;
    const uint32_t step = gridDim.x * WAVES;
    Floats<D> fk, fv;
    if (i < J.tiles) {
        const Tile T(J, i);
        fk.load(J.k.p, T.at(J.k), J.type);
        fv.load(J.v.p, T.at(J.v), J.type);
    }
    turn_rows<D>(FORWARD, SIDE, J.sa, J.sb, A);
    __syncthreads();
    uint32_t lost = 0;
    for (; i < J.tiles; i += step) {
        const Tile T(J, i);
        const int64_t pos = J.len_in[J.seq_lo + T.b] + T.t;
        uint8_t *const head = plane_ptr(g, J.seq_lo + T.b, T.h, 0);
        const bool there = T.there && pos < g.capacity;
        uint32_t wk[(D / 4 * KB + 31) / 32], wv_[(D / 4 * VB + 31) / 32], out = 0;
        const int32_t nk = append_field<D, KB>(J, J.bnd[0], fk, A, out, wk);
        if (i + step < J.tiles) {
            const Tile N(J, i + step);
            fk.load(J.k.p, N.at(J.k), J.type);
        }
        store_bits<D / 4 * KB>(g, head, 0, g.key_bytes, pos, there, wk);
        const int32_t nv = append_field<D, VB>(J, J.bnd[1], fv, A, out, wv_);
        if (i + step < J.tiles) {
            const Tile N(J, i + step);
            fv.load(J.v.p, N.at(J.v), J.type);
        }
        store_bits<D / 4 * VB>(g, head, (g.key_bytes + 15) / 16, g.value_bytes, pos, there, wv_);
        if (there && lane < 16)
            *(uint32_t *)(head + (g.n_planes - 1) * g.span + pos * 4) = ((uint32_t)nk & 0xFFFFu) | (uint32_t)nv << 16;
        lost += T.there ? out : 0;
        if (T.there && pos >= g.capacity && lane < 16)         // the host checks capacity first; this only guards memory
            atomicAdd(&J.st->fault, 1ull);
    }
    if (J.count) {
        const int64_t all = wave_sum_i64((int64_t)lost);
        if (lane == 0 && all) atomicAdd(&J.st->range_errors, (unsigned long long)all);
    }
}

// The lane's codes of a token's field of BITS-bit codes, D / 4 channels, and 16 of them as their centroids' digits.
template <int D, int BITS>
struct Field {
    Codes<D, BITS == 1 ? 2 : BITS> c;
    uint32_t w;
    __device__ __forceinline__ void load(const uint8_t *base, int64_t span, int64_t t) {
        const int grp = (threadIdx.x & 63) >> 4;
        if constexpr (BITS > 1)
            c.load(base, span, t, grp);
        else if constexpr (D == 64)
            w = *(const uint16_t *)(base + t * 8 + 2 * grp);
        else
            w = *(const uint32_t *)(base + t * 16 + 4 * grp);
    }
    __device__ __forceinline__ void digits(int b, const uint32_t (&dg)[3][4], v4i (&o)[3]) const {
        if constexpr (BITS == 4) {                     // (they come out as the even and the odd codes of each 8 in turn)
            v4i x[3];
            expand16<4>(c.bits(b, (threadIdx.x & 63) >> 4), dg, x);
#pragma unroll
            for (int l = 0; l < 3; ++l)
#pragma unroll
                for (int d = 0; d < 4; d += 2) {
                    o[l][d] = (int)perm((uint32_t)x[l][d + 1], (uint32_t)x[l][d], 0x05010400u);
                    o[l][d + 1] = (int)perm((uint32_t)x[l][d + 1], (uint32_t)x[l][d], 0x07030602u);
                }
        } else if constexpr (BITS > 1) {
            expand16<BITS>(c.bits(b, (threadIdx.x & 63) >> 4), dg, o);
        } else {
#pragma unroll
            for (int d = 0; d < 4; ++d) {              // four bits to four selectors
                const uint32_t sel = ((w >> (16 * b + 4 * d) & 15u) * 0x00204081u) & 0x01010101u;
#pragma unroll
                for (int l = 0; l < 3; ++l) o[l][d] = (int)perm(0u, dg[l][0], sel);
            }
        }
    }
};

// One field of a tile's rows, back as floating values of `type` from dst on (the lane's row).
template <int D, int BITS>
__device__ __forceinline__ void read_field(const Field<D, BITS> &f, const uint32_t (&dg)[3][4], const v4i (&A)[D / 16][D / 64], float scale,
                                           void *dst, int64_t at, int type, bool there) {
    v4i x[D / 64][3];
#pragma unroll
    for (int b = 0; b < D / 64; ++b) f.digits(b, dg, x[b]);
    const int grp = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int c0 = 0; c0 < D / 16; c0 += 2) {           // 8 channels at a time
        float y[8];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            v4i T = {0, 0, 0, 0};                      // (exact: below 128 x 2^20)
#pragma unroll
            for (int l = 2; l >= 0; --l) {
                if (l < 2) T = T << 8;
#pragma unroll
                for (int b = 0; b < D / 64; ++b) T = mma(A[c0 + c][b], x[b][l], T);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) y[4 * c + i] = product((float)T[i], scale);
        }
        if (!there) continue;
        if (type == INSITU_F32) {
            float *const to = (float *)dst + at + 16 * c0 + 4 * grp;
            *(float4 *)to = make_float4(y[0], y[1], y[2], y[3]);
            *(float4 *)(to + 16) = make_float4(y[4], y[5], y[6], y[7]);
        } else {
            uint32_t h[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                h[i] = type == INSITU_F16 ? (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)y[i])
                                          : (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)y[i]);
            *(uint4 *)((uint16_t *)dst + at + 16 * c0 + 8 * grp) = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
        }
    }
}

template <int D, int KB, int VB>
__global__ void __launch_bounds__(64 * WAVES, D == 64 ? 3 : 2) read_tiles_kernel(Tiles J, const Tables *__restrict__ tabs, int turned) {
    __shared__ uint32_t dig[2][3][4];
    __shared__ v4i A_s[D / 16][D / 64][64];
    const Geom &g = J.g;
    const int tid = threadIdx.x, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    if (tid < 32) {                                    // (no code names a centroid behind the codebook's end)
        const uint32_t z = balanced((int32_t)(tid < 16 ? tabs->kc : tabs->vc)[tid & 15]);
#pragma unroll
        for (int l = 0; l < 3; ++l) ((uint8_t *)dig[tid >> 4][l])[tid & 15] = (uint8_t)(z >> (8 * l));
    }
    const int pv = (g.key_bytes + 15) / 16;
    const uint32_t step = gridDim.x * WAVES;
    uint32_t i = blockIdx.x * WAVES + (uint32_t)wv;
    Field<D, KB> fk;                                   // (rows behind the end are the cache's own memory still)
    Field<D, VB> fv;
    uint32_t norms = 0;
    auto fetch = [&](uint32_t i) __attribute__((always_inline)) {
        const Tile T(J, i);
        const uint8_t *const head = plane_ptr(g, J.seq_lo + T.b, T.h, 0);
        fk.load(head, g.span, J.t0 + T.t);
        fv.load(head + pv * g.span, g.span, J.t0 + T.t);
        norms = *(const uint32_t *)(head + (g.n_planes - 1) * g.span + (J.t0 + T.t) * 4);
    };
    if (i < J.tiles) fetch(i);
    turn_rows<D>(turned ? INVERSE : IDENTITY, J.type == INSITU_F32 ? LANES4 : LANES8, J.sa, J.sb, A_s);
    __syncthreads();
    v4i A[D / 16][D / 64];
#pragma unroll
    for (int c = 0; c < D / 16; ++c)
#pragma unroll
        for (int b = 0; b < D / 64; ++b) A[c][b] = A_s[c][b][tid & 63];
    uint32_t dk[3][4], dv[3][4];
#pragma unroll
    for (int l = 0; l < 3; ++l)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            dk[l][j] = (uint32_t)uni32((int)dig[0][l][j]);
            dv[l][j] = (uint32_t)uni32((int)dig[1][l][j]);
        }
    const float unit = unit_of(D, turned ? 1 : 0);
    for (; i < J.tiles; i += step) {
        const Tile T(J, i);
        const bool there = T.there && J.t0 + T.t < J.len_in[J.seq_lo + T.b];
        const Field<D, KB> k = fk;
        const Field<D, VB> v = fv;
        const uint32_t n = norms;
        if (i + step < J.tiles) fetch(i + step);
        if (__ballot(there) == 0) continue;
        read_field<D, KB>(k, dk, A, (float)(int16_t)(uint16_t)n * unit, J.k.p, T.at(J.k), J.type, there);
        read_field<D, VB>(v, dv, A, (float)((int32_t)n >> 16) * unit, J.v.p, T.at(J.v), J.type, there);
    }
}

// Rows of 16 bytes' alignment, in a format that the tiles take.
bool tiles_ok(const Geom &g, const FloatRows &k, const FloatRows &v, int type, int rounds) {
    if ((g.d != 64 && g.d != 128) || g.kb < 2 || g.kb > 4 || g.vb < 1 || g.vb > 3 || g.norm_frac != 9 || rounds > 1) return false;
    const int64_t size = type == INSITU_F32 ? 4 : 2;
    int64_t bits = 0;
    for (const FloatRows *r : {&k, &v}) bits |= (int64_t)(uintptr_t)r->p | r->seq * size | r->tok * size | r->head * size;
    return (bits & 15) == 0;
}
// Keys and values of KB and VB bits at D channels
template <class F>
void by_format(const Geom &g, F &&f) {
    auto bits = [&](auto d) {
        auto keys = [&](auto kb) {
            if (g.vb == 1)
                f(d, kb, std::integral_constant<int, 1>{});
            else if (g.vb == 2)
                f(d, kb, std::integral_constant<int, 2>{});
            else
                f(d, kb, std::integral_constant<int, 3>{});
        };
        if (g.kb == 2)
            keys(std::integral_constant<int, 2>{});
        else if (g.kb == 3)
            keys(std::integral_constant<int, 3>{});
        else
            keys(std::integral_constant<int, 4>{});
    };
    if (g.d == 64)
        bits(std::integral_constant<int, 64>{});
    else
        bits(std::integral_constant<int, 128>{});
}
Tiles tiles_of(const Geom &g, const FloatRows &k, const FloatRows &v, int type, int64_t n, int seq_lo, int seq_hi, const int64_t *len,
               const RotSigns &sg) {
    Tiles J{};
    J.g = g;
    J.k = k;
    J.v = v;
    J.type = type;
    J.n = n;
    J.per = (int32_t)((n + 15) / 16);
    J.tiles = (uint32_t)J.per * (uint32_t)(seq_hi - seq_lo) * (uint32_t)g.n_kv;
    J.seq_lo = seq_lo;
    J.seq_hi = seq_hi;
    J.len_in = len;
    J.sa = sg.s0a;
    J.sb = sg.s0b;
    return J;
}
unsigned tiles_grid(int64_t tiles, int per_cu) {
    const int64_t blocks = (tiles + WAVES - 1) / WAVES;
    return (unsigned)(blocks < 256 * per_cu ? blocks : 256 * per_cu);
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
                               int rounds, const uint64_t (*signs)[2], const Tables &host, bool count, DevStats *st) {
    const int64_t rows = (int64_t)(seq_hi - seq_lo) * n_tok * g.n_kv;
    if (rows <= 0) return hipSuccess;
    if (rounds < 0 || rounds > 2) return hipErrorInvalidValue;
    const RotSigns sg = rounds ? rot_signs(rounds, signs) : RotSigns{};
    bool tiles = rounds == 1 && rows < int64_t(1) << 31 && fr::tiles_ok(g, k, v, type, rounds) && host.bnd_sorted;
    for (int i = 0; i + 1 < 1 << g.kb; ++i) tiles = tiles && std::abs(host.kbnd[i]) < 1 << 23;
    for (int i = 0; i + 1 < 1 << g.vb; ++i) tiles = tiles && std::abs(host.vbnd[i]) < 1 << 23;
    if (tiles) {
        fr::Tiles J = fr::tiles_of(g, k, v, type, n_tok, seq_lo, seq_hi, len_in, sg);
        J.len_out = len_out;
        J.len_now = len_now;
        J.count = count ? 1 : 0;
        J.st = st;
        for (int i = 0; i + 1 < 1 << g.kb; ++i) J.bnd[0][i] = (double)host.kbnd[i] * 0x1p-8;
        for (int i = 0; i + 1 < 1 << g.vb; ++i) J.bnd[1][i] = (double)host.vbnd[i] * 0x1p-8;
        fr::by_format(g, [&](auto d, auto kb, auto vb) {
            constexpr int D = decltype(d)::value, KB = decltype(kb)::value, VB = decltype(vb)::value;
            hipLaunchKernelGGL((fr::append_tiles_kernel<D, KB, VB>), dim3(fr::tiles_grid(J.tiles, D == 64 ? 4 : 2)), dim3(64 * fr::WAVES), 0, s, J);
        });
        return hipGetLastError();
    }
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
    if (rows < int64_t(1) << 31 && fr::tiles_ok(g, k, v, type, rounds)) {
        fr::Tiles J = fr::tiles_of(g, k, v, type, n, seq_lo, seq_hi, len, sg);
        J.t0 = t0;
        fr::by_format(g, [&](auto d, auto kb, auto vb) {
            constexpr int D = decltype(d)::value, KB = decltype(kb)::value, VB = decltype(vb)::value;
            hipLaunchKernelGGL((fr::read_tiles_kernel<D, KB, VB>), dim3(fr::tiles_grid(J.tiles, D == 64 ? 6 : 4)), dim3(64 * fr::WAVES), 0, s, J, t, rounds);
        });
        return hipGetLastError();
    }
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
