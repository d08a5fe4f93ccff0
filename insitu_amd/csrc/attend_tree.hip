// The attend of a tree of drafted tokens (speculative decoding): the last n rows of a sequence are the
// tree's nodes, and node i attends the context before them, its ancestors and itself, in row order, with
// the integers that attend_online / attend_two_pass (ops/attention.py:429-513) give on those rows. The
// reference decodes token by token and has no counterpart.
//
// A row of this file is one (node, query head) of a KV head's group; a wave takes tiles of 16 rows by 16
// tokens over one span of the context. Every span is walked at the same time, in three launches that
// wait on nobody:
//   max_kernel     each (row, span)'s largest score;
//   sum_kernel     the walk, from the maximum of the spans before (online) or of all (two-pass): the terms
//                  floor(v_norm p c / 2^23) of a run of rows between two events are only added, so a span
//                  gives a run's sum S and denominator L without knowing what came before it. Where the
//                  maximum rises (an event) a run ends, and the next begins with the factor f that scales
//                  what it finds: the first span, which begins with nothing, does so in place, the others
//                  hand over each run;
//   combine_kernel acc = floor(acc f / 2^15) + S, l = floor(l f / 2^15) + L over the runs in order, which is the
//                  recurrence itself as long as the clamp of acc after every token cannot fire: |acc| plus
//                  the sum of a run's |terms| below 2^31 proves that. Then acc / l.
// A row that cannot be proven (also: a query value past three digits, a score past 32 bits, a term past three
// digits, more events than the spans' runs hold) is recomputed token by token (serial_head.h).
//
// Matrix operands as in the prefill attend: scores from three balanced digits of q and of the centroids,
// nine int8 products a 64 channels, lane = (row, 4 tokens); there p and the terms of all value codes, as
// three digits, which the one-hot value codes of the tokens sum up, lane = (row, 4 channels).
#include <algorithm>
#include <cstdlib>

#include "digits.h"
#include "query.h"
#include "serial_head.h"
#include "wave.h"

namespace insitu {
namespace tr {

constexpr int W = 4;                                   // waves a workgroup of max_kernel and sum_kernel
constexpr int CW = 8;                                  // and of combine_kernel, two rows each
constexpr int UPW = TREE_NODES / 32 + 3;               // words of a node's path: ones, the bits, two of zeros
constexpr int EXTRA = 256;                             // runs a row tile holds beside its spans' first ones
constexpr int SPAN_MAX = 32768;                        // tokens a span: its events fit 31 bits, its L 32
constexpr uint32_t LUT_N = LUT_SPAN + 1;
constexpr double TERM_MAGIC = 402653184.0 + 8421504.0; // 1.5 * 2^28 + 0x808080: ulp 2^-24
constexpr double TERM_LIMIT = 8355711.0;               // 0x7F7F7F: three balanced bytes
constexpr double DOT_MAX = 0x1p46;                     // ||q||_1 max|c| below it: dot / 2^16 fits int32
constexpr double NARROW_LIMIT = 36028797018963968.0 - 16777216.0;   // |dot k_norm| below it: the score fits int32
constexpr int32_t NONE = INT32_MIN;                    // no score yet
constexpr uint32_t BAD = 1u << 31, USED = 1u << 16;

struct __attribute__((aligned(4))) u128 {              // 16 bytes of a 4-byte aligned address
    uint32_t x, y, z, w;
};

// Per row tile: 16 nspan runs, the first of each (span, row), and EXTRA more.
struct Scratch {
    int32_t *top;          // [tile][span][16]: largest scores
    uint32_t *over;        // [tile][span]: rows whose scores did not do, a bit each
    uint32_t *ev;          // [tile][span][16]: events, BAD
    uint32_t *pool;        // [tile]: extra runs taken
    uint4 *meta;           // [tile][run]: L, f | USED, the next run of the span or -1, a bound of |terms| (float)
    int32_t *S;            // [tile][run][d]
};

struct Job {
    Geom g;
    const Tables *tabs;
    const int32_t *q;
    int32_t *out;
    const int64_t *len;
    const int32_t *parents;
    int64_t pstride;
    int32_t n, rows, tiles, span, nspan, two, seq0, nseq, count;   // count: gather statistics
    Scratch sc;
    DevStats *st;
};

__device__ __forceinline__ int32_t imax(int32_t a, int32_t b) { return a > b ? a : b; }
__device__ __forceinline__ int32_t imin(int32_t a, int32_t b) { return a < b ? a : b; }
// Over a row's four lanes.
__device__ __forceinline__ int32_t row_max(int32_t v) {
    v = imax(v, __shfl_xor(v, 16));
    return imax(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ uint32_t row_or(uint32_t v) {
    v |= (uint32_t)__shfl_xor((int)v, 16);
    return v | (uint32_t)__shfl_xor((int)v, 32);
}
__device__ __forceinline__ uint32_t row_sum(uint32_t v) {
    v += (uint32_t)__shfl_xor((int)v, 16);
    return v + (uint32_t)__shfl_xor((int)v, 32);
}

// The paths of all nodes: bit 32 + j of up[i] is set where j is i or an ancestor of it; the word before
// is ones (the context's rows), those behind are zeros. Each round doubles how far a node has looked up.
// Returns the number of parents that are none (this thread's).
__device__ __forceinline__ int tree_paths(const int32_t *__restrict__ parents, int n, uint32_t (*up)[UPW], int16_t *at) {
    const int i = threadIdx.x, words = (n + 31) / 32;
    int bad = 0;
    int p = -1;
    if (i < n) {
        p = parents[i];
        bad = p >= i || p < -1;
        p = bad ? -1 : p;
        at[i] = (int16_t)p;
        for (int k = 0; k < UPW; ++k) up[i][k] = k == 0 ? ~0u : k - 1 == i >> 5 ? 1u << (i & 31) : 0u;
    }
    __syncthreads();
    while (__syncthreads_or(p >= 0)) {
        uint32_t w[UPW - 3];
        int far = -1;
        if (p >= 0) {
            far = at[p];
#pragma unroll
            for (int k = 0; k < UPW - 3; ++k) w[k] = k < words ? up[p][1 + k] : 0u;
        }
        __syncthreads();
        if (p >= 0) {
#pragma unroll
            for (int k = 0; k < UPW - 3; ++k)
                if (k < words) up[i][1 + k] |= w[k];
            at[i] = (int16_t)far;
        }
        p = far;
    }
    return bad;
}

// Which of tokens rel .. rel + 3 behind the context a row sees, a bit each (rel from -16 on).
__device__ __forceinline__ uint32_t visible4(const uint32_t *up, int rel) {
    const int k = (rel + 32) >> 5;
    return __builtin_amdgcn_alignbit(up[k + 1], up[k], rel & 31) & 15u;
}

// A row tile's queries: lane = (row, D / 4 channels from grp D / 4 on, in the order the codes expand in).
template <int D, int KB>
struct Query {
    v4i qd[3][D / 64];
    bool bad;                                          // the row needs the serial path
    bool check;                                        // scores of the tile may leave int32 (wave-uniform)
    __device__ __forceinline__ void load(const Job &J, int b, int kvh, int tile, double cmax, unsigned long long *range) {
        const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
        const int r = imin(tile * 16 + col, J.rows - 1), G = J.g.G;
        const int32_t *row = J.q + (((int64_t)b * J.n + r / G) * J.g.n_q + kvh * G + r % G) * D + grp * (D / 4);
        int64_t l1 = 0;
        uint32_t wide = 0, out = 0;
#pragma unroll
        for (int k = 0; k < D / 64; ++k) {
            uint32_t z[16];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const u128 v = *(const u128 *)(row + 16 * k + 4 * i);
                const int32_t x[4] = {(int32_t)v.x, (int32_t)v.y, (int32_t)v.z, (int32_t)v.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t a = x[j] < 0 ? 0u - (uint32_t)x[j] : (uint32_t)x[j];
                    l1 += a;
                    out += a >= (uint32_t)Q_ROT_LIMIT ? 1 : 0;
                    wide |= a > 0x7F7F7Fu ? 1u : 0u;
                    z[4 * i + j] = balanced(x[j]);
                }
            }
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                uint32_t o[3] = {0, 0, 0};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t y = z[channel_of(KB, 4 * w + j)];
#pragma unroll
                    for (int i = 0; i < 3; ++i) o[i] |= ((y >> (8 * i)) & 0xFFu) << (8 * j);
                }
#pragma unroll
                for (int i = 0; i < 3; ++i) qd[i][k][w] = (int)o[i];
            }
        }
        double b1 = (double)l1 * cmax;
        b1 += __shfl_xor(b1, 16);
        b1 += __shfl_xor(b1, 32);
        bad = row_or(wide) != 0 || !(b1 < DOT_MAX);
        check = __ballot(!bad && !(b1 * 32768.0 < NARROW_LIMIT)) != 0;
        if (range && out && tile * 16 + col < J.rows) atomicAdd(range, (unsigned long long)out);
    }
};

// A lane's share of a tile's keys as digits: token t0 + lane % 16, channels of its group.
template <int D, int KB>
struct Keys {
    Codes<D, KB> c;
    uint4 norms;                                       // of tokens t0 + 4 grp .. + 3: (k, v) int16 each
    // Rows up to the tile's end are read whatever the sequence's length: a plane holds a multiple of 256.
    __device__ __forceinline__ void load(const uint8_t *hb, const uint8_t *nb, int64_t span, int64_t t0) {
        const int lane = threadIdx.x & 63;
        c.load(hb, span, t0 + (lane & 15), lane >> 4);
        norms = *(const uint4 *)(nb + (t0 + 4 * (lane >> 4)) * 4);
    }
    __device__ __forceinline__ void expand(const uint32_t (&dg)[3][4], v4i (&a)[D / 64][3]) const {
#pragma unroll
        for (int k = 0; k < D / 64; ++k) expand16<KB>(c.bits(k, (threadIdx.x & 63) >> 4), dg, a[k]);
    }
};

// floor(dot k_norm / 2^24) of the lane's row and 4 tokens: dot = 2^16 H + L, each digit weight's sum carried
// into the next product's accumulator. Returns whether a visible one (bits of `in`) left int32.
template <int D>
__device__ __forceinline__ bool scores(const v4i (&a)[D / 64][3], const v4i (&qd)[3][D / 64], const uint4 &norms, bool check,
                                       uint32_t in, int32_t (&s)[4]) {
    v4i H = {0, 0, 0, 0}, L = {0, 0, 0, 0};
#pragma unroll
    for (int k = 4; k >= 2; --k) {
        if (k < 4) H = H << 8;
#pragma unroll
        for (int b = 0; b < D / 64; ++b)
#pragma unroll
            for (int l = 0; l < 3; ++l)
                if (k - l >= 0 && k - l < 3) H = mma(a[b][l], qd[k - l][b], H);
    }
#pragma unroll
    for (int k = 1; k >= 0; --k) {
        if (k < 1) L = L << 8;
#pragma unroll
        for (int b = 0; b < D / 64; ++b)
#pragma unroll
            for (int l = 0; l <= k; ++l) L = mma(a[b][l], qd[k - l][b], L);
    }
    const uint32_t nw[4] = {norms.x, norms.y, norms.z, norms.w};
    int64_t x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int32_t kn = (int16_t)(uint16_t)nw[i];
        x[i] = (int64_t)H[i] * kn + (((int64_t)L[i] * kn) >> 16);          // floor(dot k_norm / 2^16)
        s[i] = (int32_t)(uint32_t)((uint64_t)x[i] >> 8);
    }
    bool over = false;
    if (check) {
#pragma unroll
        for (int i = 0; i < 4; ++i) over |= ((x[i] >> 8) != (int64_t)s[i] || s[i] == NONE) && (in >> i & 1) != 0;
    }
    return over;
}

// A workgroup's place: chains fastest (a KV head's rows then stay in one XCD's cache where there are 8),
// then the row tiles, which read the same tokens, then the spans.
struct Place {
    int chain, b, kvh, tile, s;
    int64_t T, base, lo, hi;                           // the wave's span [lo, hi) of T rows
    bool tail;                                         // the workgroup's spans reach the tree's rows
    __device__ __forceinline__ bool find(const Job &J) {
        const int chains = J.nseq * J.g.n_kv;
        chain = (int)(blockIdx.x % (unsigned)chains);
        const int rest = (int)(blockIdx.x / (unsigned)chains);
        tile = rest % J.tiles;
        const int s0 = rest / J.tiles * W;
        s = s0 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        b = J.seq0 + chain / J.g.n_kv;
        kvh = chain % J.g.n_kv;
        T = J.len[b];
        base = T - J.n;
        const int64_t end = (int64_t)(s0 + W) * J.span;
        tail = (end < T ? end : T) > base;
        lo = (int64_t)s * J.span;
        hi = lo + J.span < T ? lo + J.span : T;
        return (int64_t)s0 * J.span < T;
    }
};

struct Digits {
    alignas(16) uint32_t dig[3][4];
    __device__ __forceinline__ void fill(const Tables *tabs, int kb) {
        if (threadIdx.x < 16) {
            const uint32_t z = balanced((int)threadIdx.x < (1 << kb) ? (int32_t)tabs->kc[threadIdx.x] : 0);
#pragma unroll
            for (int l = 0; l < 3; ++l) ((uint8_t *)dig[l])[threadIdx.x] = (uint8_t)(z >> (8 * l));
        }
    }
    __device__ __forceinline__ void read(uint32_t (&dg)[3][4]) const {
#pragma unroll
        for (int i = 0; i < 3; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) dg[i][j] = (uint32_t)uni32((int)dig[i][j]);
    }
};

template <int D, int KB>
__global__ void __launch_bounds__(W * 64, 4) max_kernel(Job J) {
    __shared__ Digits dgs;
    __shared__ uint32_t up[TREE_NODES][UPW];
    __shared__ int16_t at[TREE_NODES];
    Place p;
    if (!p.find(J)) return;
    const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
    dgs.fill(J.tabs, J.g.kb);
    int none = 0;
    if (p.tail) none = tree_paths(J.parents + p.b * J.pstride, J.n, up, at);
    __syncthreads();
    if (J.count && none && p.kvh == 0 && p.tile == 0 && p.T <= (int64_t)(p.s / W + 1) * W * J.span)
        atomicAdd(&J.st->range_errors, (unsigned long long)none);
    if (p.lo >= p.hi) return;
    Query<D, KB> Q;
    Q.load(J, p.b, p.kvh, p.tile, J.tabs->kc_absmax, J.count && p.s == 0 ? &J.st->range_errors : nullptr);
    uint32_t dg[3][4];
    dgs.read(dg);
    const uint8_t *hb = plane_ptr(J.g, p.b, p.kvh, 0), *nb = hb + (J.g.n_planes - 1) * J.g.span;
    const uint32_t *path = up[imin(p.tile * 16 + col, J.rows - 1) / J.g.G];
    int32_t m = NONE, lowest = 0;
    bool over = Q.bad;
    Keys<D, KB> next;
    next.load(hb, nb, J.g.span, p.lo);
    for (int64_t t0 = p.lo; t0 < p.hi; t0 += 16) {
        const Keys<D, KB> cur = next;
        if (t0 + 16 < p.hi) next.load(hb, nb, J.g.span, t0 + 16);
        v4i a[D / 64][3];
        cur.expand(dg, a);
        uint32_t in = 15u;
        if (t0 + 16 > p.base) in = visible4(path, (int)(t0 - p.base) + 4 * grp);
        int32_t s[4];
        over |= scores<D>(a, Q.qd, cur.norms, Q.check, in, s);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool on = in >> i & 1;
            m = on && s[i] > m ? s[i] : m;
            lowest = on && s[i] < lowest ? s[i] : lowest;
        }
    }
    const int64_t tl = (int64_t)p.chain * J.tiles + p.tile, at0 = tl * J.nspan + p.s;
    m = row_max(m);
    if (grp == 0) J.sc.top[at0 * 16 + col] = m;
    const uint64_t bad = __ballot(over);
    if (lane == 0) {
        J.sc.over[at0] = (uint32_t)((bad | bad >> 16 | bad >> 32 | bad >> 48) & 0xFFFFu);
        if (p.s == 0) J.sc.pool[tl] = 0;
    }
    if (J.count) {
        const bool mine = !over && p.tile * 16 + col < J.rows;
        const int64_t a = m == NONE ? 0 : m < 0 ? -(int64_t)m : m, c = -(int64_t)lowest;
        const int64_t x = wave_max_i64(mine ? (a > c ? a : c) : 0);
        if (lane == 0 && (unsigned long long)x > J.st->max_abs_score) atomicMax(&J.st->max_abs_score, (unsigned long long)x);
    }
}

// A tile's value words, lane = tokens t0 + 4 grp .. + 3; then one-hot, lane = (channel 16 c + lane % 16, 4 tokens).
template <int D, int NC>
struct Values {
    static constexpr int VW = D * (NC == 8 ? 3 : 2) / 32;
    uint32_t w[4][VW];
    __device__ __forceinline__ void load(const uint8_t *vb0, int64_t span, int64_t t0, int vb) {
        const int64_t t = t0 + 4 * ((threadIdx.x & 63) >> 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (NC == 8) {
#pragma unroll
                for (int p = 0; p < VW / 4; ++p) {
                    const uint4 v = *(const uint4 *)(vb0 + p * span + (t + i) * 16);
                    w[i][4 * p] = v.x;
                    w[i][4 * p + 1] = v.y;
                    w[i][4 * p + 2] = v.z;
                    w[i][4 * p + 3] = v.w;
                }
                if constexpr (VW % 4) {
                    const uint2 v = *(const uint2 *)(vb0 + (VW / 4) * span + (t + i) * 8);
                    w[i][VW - 2] = v.x;
                    w[i][VW - 1] = v.y;
                }
            } else if (vb == 2) {
#pragma unroll
                for (int p = 0; p < VW / 4; ++p) {
                    const uint4 v = *(const uint4 *)(vb0 + p * span + (t + i) * 16);
                    w[i][4 * p] = v.x;
                    w[i][4 * p + 1] = v.y;
                    w[i][4 * p + 2] = v.z;
                    w[i][4 * p + 3] = v.w;
                }
            } else {                                   // 1-bit codes as 2-bit ones
#pragma unroll
                for (int k = 0; k < VW; k += 4) {
                    const uint2 v = *(const uint2 *)(vb0 + (t + i) * (D / 8) + 2 * k);
                    w[i][k] = spread(v.x & 0xFFFFu);
                    w[i][k + 1] = spread(v.x >> 16);
                    w[i][k + 2] = spread(v.y & 0xFFFFu);
                    w[i][k + 3] = spread(v.y >> 16);
                }
            }
        }
    }
    static __device__ __forceinline__ uint32_t spread(uint32_t x) {
        x = (x | x << 8) & 0x00FF00FFu;
        x = (x | x << 4) & 0x0F0F0F0Fu;
        x = (x | x << 2) & 0x33333333u;
        return (x | x << 1) & 0x55555555u;
    }
    __device__ __forceinline__ void onehot(int c, int col, v4i (&oh)[NC / 4]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (NC == 4) {
                oh[0][i] = (int)(1u << (8 * (w[i][c] >> (2 * col) & 3u)));
            } else {
                // 16 channels are 48 bits, from bit 0 of word 3 c / 2 or bit 16 of the word before its end
                const int w0 = 48 * c / 32, sh = 48 * c % 32 + 3 * col;
                const uint32_t hi = w[i][w0 + 1], lo = sh < 32 ? w[i][w0] : hi;
                const uint64_t h = 1ull << (8 * (__builtin_amdgcn_alignbit(hi, lo, sh & 31) & 7u));
                oh[i >> 1][2 * (i & 1)] = (int)(uint32_t)h;
                oh[i >> 1][2 * (i & 1) + 1] = (int)(uint32_t)(h >> 32);
            }
        }
    }
};

template <int D, int KB, int NC>
__global__ void __launch_bounds__(W * 64, D == 64 && NC == 4 ? 3 : 2) sum_kernel(Job J) {
    constexpr int CT = D / 16, PVK = NC / 4;
    __shared__ Digits dgs;
    __shared__ uint32_t up[TREE_NODES][UPW];
    __shared__ int16_t at[TREE_NODES];
    __shared__ uint16_t lut_s[LUT_N + 7];
    Place p;
    if (!p.find(J)) return;
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, grp = lane >> 4;
    dgs.fill(J.tabs, J.g.kb);
    {
        const int32_t x = J.tabs->exp_table[tid];
#pragma unroll
        for (int i = 0; i < LUT_SPAN / 256; ++i) lut_s[256 * i + tid] = (uint16_t)(x >> i);
        if (tid == 0) lut_s[LUT_SPAN] = 0;
    }
    if (p.tail) tree_paths(J.parents + p.b * J.pstride, J.n, up, at);
    __syncthreads();
    if (p.lo >= p.hi) return;

    const int64_t tl = (int64_t)p.chain * J.tiles + p.tile;
    // the maximum of the spans before, or of all
    int32_t m = NONE;
    {
        const int end = J.two ? (int)((p.T + J.span - 1) / J.span) : p.s;
        const int32_t *top = J.sc.top + tl * J.nspan * 16 + col;
        for (int i = grp; i < end; i += 4) m = imax(m, top[i * 16]);
        m = row_max(m);
    }
    Query<D, KB> Q;
    Q.load(J, p.b, p.kvh, p.tile, J.tabs->kc_absmax, nullptr);
    uint32_t dg[3][4];
    dgs.read(dg);
    double vcs[NC], vcmax = 0.0;                       // value centroids / 2^23
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        vcs[i] = __longlong_as_double(uni64(__double_as_longlong(i < (1 << J.g.vb) ? (double)J.tabs->vc[i] * 0x1p-23 : 0.0)));
        vcmax = fmax(vcmax, fabs(vcs[i]));
    }
    const uint32_t delta_max = (uint32_t)J.tabs->delta_max;
    const uint8_t *hb = plane_ptr(J.g, p.b, p.kvh, 0), *nb = hb + (J.g.n_planes - 1) * J.g.span;
    const uint8_t *vb0 = hb + (int64_t)((J.g.key_bytes + 15) / 16) * J.g.span;
    const uint32_t *path = up[imin(p.tile * 16 + col, J.rows - 1) / J.g.G];
    const int vb = J.g.vb;
    const bool first = p.s == 0;                       // what the span finds is nothing: it scales in place
    const int64_t run0 = tl * (16 * (int64_t)J.nspan + EXTRA);

    v4i acc[CT];                                       // lane = (row, 4 channels of each 16)
#pragma unroll
    for (int c = 0; c < CT; ++c) acc[c] = v4i{0, 0, 0, 0};
    uint32_t lp = 0;                                   // the lane's part of the denominator since the last event
    uint32_t l0 = 0;                                   // first span: the row's denominator up to there
    float bs = 0.0f;                                   // the lane's part of sum |v_norm p|
    uint32_t wmax = 0;                                 // its largest
    uint32_t n_ev = 0;                                 // the lane's events
    bool bad = Q.bad;
    int slot = p.s * 16 + col;                         // the row's open run, and its factor
    uint32_t fopen = 1u << PROB_FRAC;

    auto lut = [&](uint32_t d) __attribute__((always_inline)) -> uint32_t {
        return lut_s[__umulhi(d, (uint32_t)LOG2E_Q16 << 8)];        // floor(d log2(e) / 2^24), d <= delta_max
    };
    auto clip = [&](int32_t hi, int32_t lo) __attribute__((always_inline)) -> uint32_t {
        const uint32_t w = (uint32_t)hi - (uint32_t)lo;
        return w < delta_max ? w : delta_max;
    };
    auto accumulate = [&](const v4i (&A)[3][PVK], const Values<D, NC> &V) __attribute__((always_inline)) {
        // (opaque, so that the one-hot codes are made where they are used: kept over an events' loop they
        // take 16 to 64 registers)
        int ch = col;
        asm volatile("" : "+v"(ch));
#pragma unroll
        for (int c = 0; c < CT; ++c) {
            v4i oh[PVK], t = {0, 0, 0, 0};
            V.onehot(c, ch, oh);
#pragma unroll
            for (int k = 0; k < PVK; ++k) t = mma(oh[k], A[2][k], t);
            t = t << 8;
#pragma unroll
            for (int k = 0; k < PVK; ++k) t = mma(oh[k], A[1][k], t);
            t = (t << 8) + acc[c];
#pragma unroll
            for (int k = 0; k < PVK; ++k) t = mma(oh[k], A[0][k], t);
            acc[c] = t;
        }
    };
    // the open run of the rows where `has`: into its record
    auto hand_over = [&](bool has, int next) __attribute__((always_inline)) {
        const uint32_t L = row_sum(lp);
        float b = bs;
        b += __shfl_xor(b, 16);
        b += __shfl_xor(b, 32);
        if (!has) return;
        const bool used = L != 0 || fopen != 1u << PROB_FRAC;
        if (grp == 0)
            J.sc.meta[run0 + slot] = make_uint4(L, fopen | (used ? USED : 0u), (uint32_t)next,
                                                __float_as_uint(b * (float)vcmax * 1.001f + (float)J.span));
        if (!used) return;
        int32_t *to = J.sc.S + (run0 + slot) * D + 4 * grp;
#pragma unroll
        for (int c = 0; c < CT; ++c) *(v4i *)(to + 16 * c) = acc[c];
    };

    Keys<D, KB> nxt;
    nxt.load(hb, nb, J.g.span, p.lo);
    for (int64_t t0 = p.lo; t0 < p.hi; t0 += 16) {
        const Keys<D, KB> cur = nxt;
        Values<D, NC> V;
        V.load(vb0, J.g.span, t0, vb);
        if (t0 + 16 < p.hi) nxt.load(hb, nb, J.g.span, t0 + 16);
        v4i a[D / 64][3];
        cur.expand(dg, a);
        const bool tail = t0 + 16 > p.base;
        uint32_t in = 15u;
        if (tail) in = visible4(path, (int)(t0 - p.base) + 4 * grp);
        int32_t s[4];
        scores<D>(a, Q.qd, cur.norms, false, in, s);
        if (tail) {
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] = in >> i & 1 ? s[i] : NONE;
        }
        const int32_t mx = imax(imax(s[0], s[1]), imax(s[2], s[3]));
        const uint64_t evl = __ballot(mx > m);
        if (evl == 0 && __ballot((uint32_t)m - (uint32_t)mx < delta_max) == 0) continue;      // every p is 0
        const uint32_t nw[4] = {cur.norms.x, cur.norms.y, cur.norms.z, cur.norms.w};
        v4i A[3][PVK];
        uint32_t pw[4];
        auto weights = [&](const uint32_t (&dl)[4]) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < 4; ++i) pw[i] = lut(dl[i]);
            if (tail) {
#pragma unroll
                for (int i = 0; i < 4; ++i) pw[i] = in >> i & 1 ? pw[i] : 0u;
            }
        };
        // the terms of every (token, code) as digit bytes, of the tokens of segment `sg` (of seg). NC = 4: dword =
        // token; NC = 8: block = token pair, dword = (token, half its codes)
        auto terms = [&](uint32_t seg, uint32_t sg) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t pi = ((seg >> (8 * i)) & 0xFFu) == sg ? pw[i] : 0u;
                lp += pi;
                const int32_t w = __mul24((int32_t)nw[i] >> 16, (int)pi);
            const uint32_t aw = w < 0 ? 0u - (uint32_t)w : (uint32_t)w;
                wmax = aw > wmax ? aw : wmax;
                bs += (float)aw;
                const double wd = (double)w;
#pragma unroll
                for (int k4 = 0; k4 < NC / 4; ++k4) {
                    const int kbk = NC == 4 ? 0 : i >> 1, dw = NC == 4 ? i : 2 * (i & 1) + k4;
                    uint32_t yl[4], yh[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint64_t y = (uint64_t)__double_as_longlong(fma(wd, vcs[4 * k4 + k], TERM_MAGIC));
                        yl[k] = (uint32_t)y;
                        yh[k] = (uint32_t)(y >> 32);
                    }
                    const uint32_t l01 = perm(yl[1], yl[0], 0x0C0C0703u), l23 = perm(yl[3], yl[2], 0x07030C0Cu);
                    const uint32_t h01 = perm(yh[1], yh[0], 0x05010400u), h23 = perm(yh[3], yh[2], 0x05010400u);
                    A[0][kbk][dw] = (int)((l01 | l23) ^ 0x80808080u);
                    A[1][kbk][dw] = (int)(perm(h23, h01, 0x05040100u) ^ 0x80808080u);
                    A[2][kbk][dw] = (int)(perm(h23, h01, 0x07060302u) ^ 0x80808080u);
                }
            }
        };
        if (evl == 0) {
            const uint32_t dl[4] = {clip(m, s[0]), clip(m, s[1]), clip(m, s[2]), clip(m, s[3])};
            weights(dl);
            terms(0u, 0u);
            accumulate(A, V);
            continue;
        }
        // events: the row's tokens fall into segments, one more than its events (bits 8 i of seg the
        // segment of token i)
        int32_t e = m;                                 // the maximum before the lane's tokens
        {
            const int32_t x = __shfl(mx, lane - 16), y = __shfl(mx, lane - 32), z = __shfl(mx, lane - 48);
            if (grp > 0) e = imax(e, x);
            if (grp > 1) e = imax(e, y);
            if (grp > 2) e = imax(e, z);
        }
        uint32_t dl[4], fe[4], seg = 0, n = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool ev = s[i] > e;
            const uint32_t dd = clip(ev ? s[i] : e, ev ? e : s[i]);
            fe[i] = ev ? dd + 1u : 0u;                 // an event's distance, + 1
            dl[i] = ev ? 0u : dd;
            e = ev ? s[i] : e;
            n += ev ? 1 : 0;
            seg |= n << (8 * i);
        }
        const uint32_t n1 = (uint32_t)__shfl((int)n, lane - 16), n2 = (uint32_t)__shfl((int)n, lane - 32),
                       n3 = (uint32_t)__shfl((int)n, lane - 48);
        const uint32_t off = (grp > 0 ? n1 : 0) + (grp > 1 ? n2 : 0) + (grp > 2 ? n3 : 0);
        seg += off * 0x01010101u;                      // at most 16
        const int row_ev = __shfl((int)(off + n), 48 + col);
        m = __shfl(e, 48 + col);
        n_ev += n;
        weights(dl);
        for (int sg = 0;; ++sg) {
            terms(seg, (uint32_t)sg);
            accumulate(A, V);
            const bool has = row_ev > sg;
            if (__ballot(has) == 0) break;
            // the event that opens segment sg + 1 of the row
            uint32_t fd = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) fd = ((seg >> (8 * i)) & 0xFFu) == (uint32_t)(sg + 1) && fe[i] ? fe[i] : fd;
            fd = row_or(fd);
            const uint32_t f = has ? lut(fd - 1u) : 1u << PROB_FRAC;
            if (first) {
#pragma unroll
                for (int c = 0; c < CT; ++c)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[c][i] = (int32_t)(((int64_t)acc[c][i] * (int32_t)f) >> PROB_FRAC);
                const uint32_t l = l0 + row_sum(lp);
                if (has) {
                    l0 = (uint32_t)(((uint64_t)l * f) >> PROB_FRAC);
                    lp = 0;
                }
            } else {
                int to = 0;
                if (has && grp == 0) to = (int)atomicAdd(J.sc.pool + tl, 1u);
                to = __shfl(to, col);
                bad = bad || (has && to >= EXTRA);
                to = 16 * J.nspan + imin(to, EXTRA - 1);
                hand_over(has, to);
                if (has) {
                    slot = to;
                    fopen = f;
                    lp = 0;
                    bs = 0.0f;
#pragma unroll
                    for (int c = 0; c < CT; ++c) acc[c] = v4i{0, 0, 0, 0};
                }
            }
        }
    }
    // (the first span's l0 is the same in the row's lanes)
    lp += grp == 0 ? l0 : 0u;
    hand_over(true, -1);
    bad = bad || !((double)wmax * vcmax + 2.0 <= TERM_LIMIT);
    const uint32_t events = row_sum(n_ev);
    const uint32_t any = row_or(bad ? BAD : 0u);
    if (grp == 0) J.sc.ev[(tl * J.nspan + p.s) * 16 + col] = events | any;
}

template <int D>
__global__ void __launch_bounds__(CW * 64) combine_kernel(Job J) {
    constexpr int CPL = D / 64, RS = D == 64 ? 60 : 116;
    __shared__ SerialLds<RS> fb[CW];
    __shared__ uint32_t up[CW][TREE_NODES / 32];
    __shared__ unsigned long long s_ev, s_bad, s_ovf, s_acc;
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int chains = J.nseq * J.g.n_kv;
    const int chain = (int)(blockIdx.x % (unsigned)chains), tile = (int)(blockIdx.x / (unsigned)chains);
    const int b = J.seq0 + chain / J.g.n_kv, kvh = chain % J.g.n_kv, G = J.g.G;
    const int64_t T = J.len[b], base = T - J.n, tl = (int64_t)chain * J.tiles + tile;
    const int ns = (int)((T + J.span - 1) / J.span);
    const int64_t run0 = tl * (16 * (int64_t)J.nspan + EXTRA);
    if (tid == 0) s_ev = s_bad = s_ovf = s_acc = 0;
    __syncthreads();
    for (int col = wv; col < 16; col += CW) {
        const int r = tile * 16 + col;
        if (r >= J.rows) break;
        const int node = r / G;
        const int64_t qrow = (((int64_t)b * J.n + node) * J.g.n_q + kvh * G + r % G) * D;
        int64_t acc[CPL], l = 0;
#pragma unroll
        for (int k = 0; k < CPL; ++k) acc[k] = 0;
        uint32_t events = 0;
        bool bad = false;
        for (int i0 = 0; i0 < ns; i0 += 64) {
            const bool in = i0 + lane < ns;
            const uint32_t e = in ? J.sc.ev[(tl * J.nspan + i0 + lane) * 16 + col] : 0u;
            const uint32_t o = in ? J.sc.over[tl * J.nspan + i0 + lane] : 0u;
            events += e & ~BAD;
            bad = bad || __ballot((e & BAD) != 0 || (o >> col & 1) != 0) != 0;
        }
        for (int i0 = 0; i0 < ns && !bad; i0 += 64) {
            const uint4 mt = i0 + lane < ns ? J.sc.meta[run0 + (i0 + lane) * 16 + col] : make_uint4(0u, 0u, ~0u, 0u);
            uint64_t todo = __ballot((mt.y & USED) != 0 || mt.z != ~0u);
            constexpr int AHEAD = 4;
            int32_t v[AHEAD][CPL];
            while (todo && !bad) {
                int at[AHEAD];
                uint64_t left = todo;
#pragma unroll
                for (int j = 0; j < AHEAD; ++j) {
                    at[j] = left ? __ffsll((long long)left) - 1 : -1;
                    left &= left - 1;
                    if (at[j] < 0) continue;
                    const int32_t *S = J.sc.S + (run0 + (i0 + at[j]) * 16 + col) * D;
                    const bool used = ((uint32_t)__builtin_amdgcn_readlane((int)mt.y, at[j]) & USED) != 0;
#pragma unroll
                    for (int k = 0; k < CPL; ++k) v[j][k] = used ? S[lane + 64 * k] : 0;
                }
                todo = left;
#pragma unroll
                for (int j = 0; j < AHEAD; ++j) {
                    if (at[j] < 0) continue;
                    uint32_t L = (uint32_t)__builtin_amdgcn_readlane((int)mt.x, at[j]);
                    uint32_t f = (uint32_t)__builtin_amdgcn_readlane((int)mt.y, at[j]);
                    int next = __builtin_amdgcn_readlane((int)mt.z, at[j]);
                    double bound = (double)__uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)mt.w, at[j]));
                    for (;;) {
                        if (f & USED) {
                            const int64_t ff = f & (USED - 1);
#pragma unroll
                            for (int k = 0; k < CPL; ++k) {
                                acc[k] = (acc[k] * ff) >> PROB_FRAC;
                                const int64_t m = acc[k] < 0 ? -acc[k] : acc[k];
                                // two-pass clamps once, at the end: only the run's own sum must fit
                                bad = bad || !((J.two ? 0.0 : (double)m) + bound <= 2147483647.0);
                                acc[k] += v[j][k];
                            }
                            l = ((l * ff) >> PROB_FRAC) + L;
                        }
                        if (next < 0) break;
                        const uint4 x = J.sc.meta[run0 + next];
                        const int32_t *S = J.sc.S + (run0 + next) * D;
                        L = x.x;
                        f = x.y;
                        bound = (double)__uint_as_float(x.w);
#pragma unroll
                        for (int k = 0; k < CPL; ++k) v[j][k] = f & USED ? S[lane + 64 * k] : 0;
                        next = (int)x.z;
                    }
                }
                bad = __ballot(bad) != 0;
            }
        }
        if (bad) {
            tree_path(J.parents + b * J.pstride, node, J.n, up[wv]);
            serial_head<CPL, RS>(J.g, J.tabs, J.tabs->kc, J.tabs->vc, J.q + qrow, b, kvh, T, J.two, true, fb[wv], J.out + qrow,
                                 J.st, TreeRows{up[wv], base});
            if (lane == 0) atomicAdd(&s_bad, 1ull);
            continue;
        }
        const Recip rc = reciprocal(l);
        int64_t amax = 0, ovf = 0;
#pragma unroll
        for (int k = 0; k < CPL; ++k) {
            if (acc[k] < ACC_LO || acc[k] > ACC_HI) {
                ++ovf;
                acc[k] = acc[k] < ACC_LO ? ACC_LO : ACC_HI;
            }
            J.out[qrow + lane + 64 * k] = (int32_t)(wmul(acc[k], rc.r) >> rc.shift);
            const int64_t m = acc[k] < 0 ? -acc[k] : acc[k];
            amax = m > amax ? m : amax;
        }
        if (J.count) {
            const int64_t ev = wave_sum_i64((int64_t)events);
            amax = wave_max_i64(amax);
            ovf = wave_sum_i64(ovf);
            if (lane == 0) {
                if (ev && !J.two) atomicAdd(&s_ev, (unsigned long long)ev);
                if (ovf) atomicAdd(&s_ovf, (unsigned long long)ovf);
                atomicMax(&s_acc, (unsigned long long)amax);
            }
        }
    }
    if (!J.count) return;
    __syncthreads();
    if (tid == 0) {
        if (s_ev) atomicAdd(&J.st->rescale_events, s_ev);
        if (s_bad) atomicAdd(&J.st->serial_fallbacks, s_bad);
        if (s_ovf) atomicAdd(&J.st->acc_overflows, s_ovf);
        if (s_acc > J.st->max_abs_acc) atomicMax(&J.st->max_abs_acc, s_acc);
        if (tile == 0 && kvh == 0) atomicMax(&J.st->n_tokens, (unsigned long long)T);
    }
}

// Any format, token by token: a wave a row.
constexpr int SERIAL_RS = 272;   // >= the widest row (8b/8b at d = 128: 260 B)
template <int CPL>
__global__ void __launch_bounds__(64) serial_kernel(Job J) {
    __shared__ int64_t kc[256], vc[256];
    __shared__ __align__(16) SerialLds<SERIAL_RS> L;
    __shared__ uint32_t up[TREE_NODES / 32];
    const int lane = threadIdx.x;
    const int qh = (int)(blockIdx.x % (unsigned)J.g.n_q);
    const int64_t rest = blockIdx.x / (unsigned)J.g.n_q;
    const int node = (int)(rest % J.n), b = (int)(rest / J.n);
    const int32_t *parents = J.parents + b * J.pstride;
    for (int i = lane; i < (1 << J.g.kb); i += 64) kc[i] = J.tabs->kc[i];
    for (int i = lane; i < (1 << J.g.vb); i += 64) vc[i] = J.tabs->vc[i];
    const int64_t at = (int64_t)blockIdx.x * J.g.d;
    for (int c = lane; c < J.g.d; c += 64) {
        const int64_t x = J.q[at + c];
        if (x >= Q_ROT_LIMIT || x <= -Q_ROT_LIMIT) atomicAdd(&J.st->range_errors, 1ull);
    }
    if (qh == 0 && lane == 0 && (parents[node] >= node || parents[node] < -1)) atomicAdd(&J.st->range_errors, 1ull);
    __syncthreads();
    tree_path(parents, node, J.n, up);
    const int64_t T = J.len[b];
    serial_head<CPL, SERIAL_RS>(J.g, J.tabs, kc, vc, J.q + at, b, qh / J.g.G, T, J.two, true, L, J.out + at, J.st,
                                TreeRows{up, T - J.n});
}

// The scratch of a launch over nseq sequences, carved from p (null: only its size).
size_t carve(const Geom &g, int64_t nseq, int64_t tiles, int64_t nspan, uint8_t *p, Scratch *sc) {
    size_t o = 0;
    auto take = [&](size_t n) {
        uint8_t *a = p ? p + o : nullptr;
        o += (n + 255) / 256 * 256;
        return a;
    };
    const size_t all = (size_t)nseq * g.n_kv * tiles, runs = all * (16 * (size_t)nspan + EXTRA);
    Scratch c{};
    c.top = (int32_t *)take(all * nspan * 64);
    c.over = (uint32_t *)take(all * nspan * 4);
    c.ev = (uint32_t *)take(all * nspan * 64);
    c.pool = (uint32_t *)take(all * 4);
    c.meta = (uint4 *)take(runs * 16);
    c.S = (int32_t *)take(runs * g.d * 4);
    if (sc) *sc = c;
    return o;
}

// Sequences a launch takes, and the spans of the longest.
struct Plan {
    int64_t seqs, tiles, span, nspan;
};
constexpr size_t BUDGET = (size_t)512 << 20;
Plan plan(const Geom &g, int64_t n, int64_t longest, int64_t batch) {
    Plan p{};
    p.tiles = (n * g.G + 15) / 16;
    p.seqs = batch;
    for (;;) {
        const int64_t all = p.seqs * g.n_kv * p.tiles;
        int64_t want = (4096 + all - 1) / all, most = (longest + 63) / 64;
        const int64_t least = (longest + SPAN_MAX - 1) / SPAN_MAX;
        want = want > most ? most : want;
        want = want < least ? least : want;
        p.span = ((longest + want - 1) / want + 15) / 16 * 16;
        p.nspan = (longest + p.span - 1) / p.span;
        if (p.seqs == 1 || carve(g, p.seqs, p.tiles, p.nspan, nullptr, nullptr) <= BUDGET) return p;
        p.seqs = (p.seqs + 1) / 2;
    }
}

template <int D, int KB, int NC>
hipError_t launch(hipStream_t s, const Job &J, LaunchEv ev) {
    const int64_t chains = (int64_t)J.nseq * J.g.n_kv;
    const dim3 grid((unsigned)(chains * J.tiles * ((J.nspan + W - 1) / W)));
    hipExtLaunchKernelGGL((max_kernel<D, KB>), grid, dim3(W * 64), 0, s, ev.start, nullptr, 0, J);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipExtLaunchKernelGGL((sum_kernel<D, KB, NC>), grid, dim3(W * 64), 0, s, nullptr, nullptr, 0, J);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipExtLaunchKernelGGL((combine_kernel<D>), dim3((unsigned)(chains * J.tiles)), dim3(CW * 64), 0, s, nullptr, ev.stop, 0, J);
    return hipGetLastError();
}

}  // namespace tr

bool tree_supported(const Geom &g) {
    return (g.d == 64 || g.d == 128) && g.kb >= 2 && g.kb <= 4 && g.vb >= 1 && g.vb <= 3 && g.norm_frac == 9;
}

size_t tree_scratch_bytes(const Geom &g, int64_t n, int64_t longest) {
    const tr::Plan p = tr::plan(g, n, longest, g.batch);
    return tr::carve(g, p.seqs, p.tiles, p.nspan, nullptr, nullptr);
}

hipError_t launch_attend_tree(hipStream_t s, const Geom &g, const Tables *t, const int32_t *q, int32_t *out,
                              const int64_t *len, const int32_t *parents, int64_t pstride, int32_t n, int64_t longest,
                              int two_pass, bool count, void *scratch, size_t scratch_bytes, LaunchEv ev, DevStats *st) {
    using namespace tr;
    const Plan p = plan(g, n, longest, g.batch);
    Job J{};
    if (carve(g, p.seqs, p.tiles, p.nspan, (uint8_t *)scratch, &J.sc) > scratch_bytes) return hipErrorInvalidValue;
    J.g = g;
    J.tabs = t;
    J.q = q;
    J.out = out;
    J.len = len;
    J.parents = parents;
    J.pstride = pstride;
    J.n = n;
    J.rows = n * g.G;
    J.tiles = (int32_t)p.tiles;
    J.span = (int32_t)p.span;
    J.nspan = (int32_t)p.nspan;
    J.two = two_pass;
    J.count = count;
    J.st = st;
    for (int64_t b = 0; b < g.batch; b += p.seqs) {
        J.seq0 = (int32_t)b;
        J.nseq = (int32_t)std::min<int64_t>(p.seqs, g.batch - b);
        const LaunchEv e{b == 0 ? ev.start : nullptr, b + p.seqs >= g.batch ? ev.stop : nullptr};
        hipError_t rc = hipErrorInvalidValue;
#define INSITU_TREE_CASE(DD, KK, CC) \
    if (g.d == DD && g.kb == KK && (g.vb <= 2 ? 4 : 8) == CC) rc = launch<DD, KK, CC>(s, J, e);
#define INSITU_TREE_D(DD)                                                                              \
    INSITU_TREE_CASE(DD, 2, 4) INSITU_TREE_CASE(DD, 3, 4) INSITU_TREE_CASE(DD, 4, 4)                   \
    INSITU_TREE_CASE(DD, 2, 8) INSITU_TREE_CASE(DD, 3, 8) INSITU_TREE_CASE(DD, 4, 8)
        INSITU_TREE_D(64)
        INSITU_TREE_D(128)
#undef INSITU_TREE_D
#undef INSITU_TREE_CASE
        if (rc != hipSuccess) return rc;
    }
    return hipSuccess;
}

hipError_t launch_attend_tree_serial(hipStream_t s, const Geom &g, const Tables *t, const int32_t *q, int32_t *out,
                                     const int64_t *len, const int32_t *parents, int64_t pstride, int32_t n,
                                     int two_pass, LaunchEv ev, DevStats *st) {
    tr::Job J{};
    J.g = g;
    J.tabs = t;
    J.q = q;
    J.out = out;
    J.len = len;
    J.parents = parents;
    J.pstride = pstride;
    J.n = n;
    J.two = two_pass;
    J.st = st;
    const int64_t blocks = (int64_t)g.batch * n * g.n_q;
    if (blocks > 0x7fffffff) return hipErrorInvalidValue;
    if (g.d <= 64)
        hipExtLaunchKernelGGL(tr::serial_kernel<1>, dim3((unsigned)blocks), dim3(64), 0, s, ev.start, ev.stop, 0, J);
    else
        hipExtLaunchKernelGGL(tr::serial_kernel<2>, dim3((unsigned)blocks), dim3(64), 0, s, ev.start, ev.stop, 0, J);
    return hipGetLastError();
}

}  // namespace insitu
