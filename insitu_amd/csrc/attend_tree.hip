// The attend of a tree of drafted tokens (speculative decoding): the last n rows of a sequence are the
// tree's nodes, and node i attends the context before them, its ancestors and itself, in row order, with
// the integers that attend_online / attend_two_pass (ops/attention.py:429-513) give on those rows. The
// reference decodes token by token and has no counterpart.
//
// A row of this file is one (node, query head) of a KV head's group; a wave takes tiles of 16 rows by 16
// tokens over one span of the context. Every span is walked at the same time, in three launches that
// wait on nobody:
//   max_kernel     each row's largest score in parts of the spans;
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
//
// A context of up to 512 tokens takes one launch (fused_kernel): a workgroup's eight waves are the spans, and the
// three steps follow each other behind barriers, the runs mostly in shared memory.
//
// What bounds it. Memory does not: 32 nodes of 4 heads behind 8 x 32,768 tokens read 218 MB, 46 us at the rate of a
// copy, and take 1,770 us. The integers do, though no one unit is full: a tile of 16 x 16 at d = 128 with 3-bit values
// costs 580 vector instructions, 54 of them matrix ones, which fill 69 % of the issue slots (the matrix cores are busy
// for 26 %), and two waves a SIMD do not cover the rest, the latency of their chains: the keys' digits, the scores'
// carries in 64 bits, the terms in float64 for every value code (exact: 53 bits), their digits' bytes and the one-hot
// codes. So the tile's terms use two digits where they fit, no tile is walked whose weights are all zero (scored it is,
// once more), and max_kernel's row tiles share the expanded keys. Registers: the walk takes 201 to 256, and at d = 128
// with 3-bit values spills 11 (17 in one launch); three waves a SIMD at d = 64 spill 21 to 33, still the faster way.
// Measured kernels: 26 nodes behind 32,768 tokens (4b/2b, 32 heads) 40 + 66 + 13 us, 64 nodes behind 4,097 two-pass
// 16 + 38 + 6 us; tried and slower: 32 tokens a step, storing the scores between the launches, one launch for long
// contexts, signed codebooks halved by symmetry, two or four tokens' tiles sharing one-hot codes at d = 128
// (registers), four waves a SIMD.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "digits.h"
#include "query.h"
#include "serial_head.h"
#include "wave.h"

namespace insitu {
namespace tr {

constexpr int W = 4;                                   // waves a workgroup of max_kernel and sum_kernel
constexpr int CW = 8;                                  // and of combine_kernel, a row each
constexpr int UPW = TREE_NODES / 32 + 3;               // words of a node's path: ones, the bits, two of zeros
// runs a row tile holds beside its spans' first ones: 256, and up to 4,096 where few tiles leave room
constexpr int EXTRA_MIN = 256, EXTRA_MAX = 4096;
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

// Per row tile: 16 nspan runs, the first of each (span, row), and `extra` more.
struct Scratch {
    int32_t *top;          // [tile][max_kernel's span][16]: largest scores
    uint32_t *over;        // [tile][max_kernel's span]: rows whose scores did not do, a bit each
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
    int32_t n, rows, tiles, span, nspan, mspan, nms;   // mspan, nms: max_kernel's spans, whole parts of the others
    int32_t extra, two, seq0, nseq, count;             // count: gather statistics
    int64_t longest;
    double kc_absmax, vcs[8], vcmax;                   // ValueTable's, and its wide and delta_max
    uint32_t wide, delta_max;
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
// is ones (the context's rows), those behind are zeros. Each round doubles how far a node has looked up. p: the
// thread's node's parent, or -1. Returns the number of parents that are none (this thread's).
__device__ __forceinline__ int tree_paths(int p, int n, uint32_t (*up)[UPW], int16_t *at) {
    const int i = threadIdx.x, words = (n + 31) / 32;
    int bad = 0;
    if (i < n) {
        bad = p >= i || p < -1;
        p = bad ? -1 : p;
    }
    if (n <= 64) {                                     // one wave, in registers; the caller's barrier shows it
        if (i < 64) {
            uint32_t lo = i < 32 ? 1u << i : 0u, hi = i < 32 ? 0u : 1u << (i - 32);
            while (__ballot(p >= 0) != 0) {
                const int j = p >= 0 ? p : i;
                const uint32_t l = (uint32_t)__shfl((int)lo, j), h = (uint32_t)__shfl((int)hi, j);
                const int far = __shfl(p, j);
                lo |= l;
                hi |= h;
                p = far;
            }
            if (i < n) {
                up[i][0] = ~0u;
                up[i][1] = lo;
                up[i][2] = hi;
                up[i][3] = up[i][4] = up[i][5] = 0u;
            }
        }
        return bad;
    }
    if (i < n) {
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

// A sequence's rows. A call replayed from a graph after the lengths changed stays within the spans it was
// planned with.
__device__ __forceinline__ int64_t rows_of(const Job &J, int b) {
    const int64_t T = J.len[b] < J.longest ? J.len[b] : J.longest;
    return T < J.n ? J.n : T;
}
// Which of tokens rel .. rel + 3 behind the context a row sees, a bit each (rel from -16 on).
__device__ __forceinline__ uint32_t visible4(const uint32_t *up, int rel) {
    const int k = (rel + 32) >> 5;
    return __builtin_amdgcn_alignbit(up[k + 1], up[k], rel & 31) & 15u;
}

// A workgroup's place: chains fastest (a KV head's rows then stay in one XCD's cache where there are 8),
// then the row tiles (or groups of them), which read the same tokens, then the spans.
struct Place {
    int chain, b, kvh, tile, s;
    int64_t T, base, lo, hi;                           // the wave's span [lo, hi) of T rows
    bool tail;                                         // the workgroup's spans reach the tree's rows
    __device__ __forceinline__ bool find(const Job &J, int tiles, int span, int waves) {
        const int chains = J.nseq * J.g.n_kv;
        chain = (int)(blockIdx.x % (unsigned)chains);
        const int rest = (int)(blockIdx.x / (unsigned)chains);
        tile = rest % tiles;
        const int s0 = rest / tiles * waves;
        s = s0 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        b = J.seq0 + chain / J.g.n_kv;
        kvh = chain % J.g.n_kv;
        T = rows_of(J, b);
        base = T - J.n;
        const int64_t end = (int64_t)(s0 + waves) * span;
        tail = (end < T ? end : T) > base;
        lo = (int64_t)s * span;
        hi = lo + span < T ? lo + span : T;
        return (int64_t)s0 * span < T;
    }
};

__device__ __forceinline__ uint32_t magnitude(int32_t x) { return x < 0 ? 0u - (uint32_t)x : (uint32_t)x; }

// A row tile's queries: lane = (row, D / 4 channels from grp D / 4 on, in the order the codes expand in).
template <int D, int KB>
struct Query {
    v4i qd[3][D / 64];
    bool bad;                                          // the row needs the serial path
    bool check;                                        // scores of the tile may leave int32 (wave-uniform)
    u128 raw[4 * (D / 64)];
    int64_t at;                                        // of the lane's channels
    // the loads, and then what is made of them
    __device__ __forceinline__ void fetch(const Job &J, const Place &p, int tile) {
        const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
        const int r = imin(tile * 16 + col, J.rows - 1), G = J.g.G;
        at = (((int64_t)p.b * J.n + r / G) * J.g.n_q + p.kvh * G + r % G) * D + grp * (D / 4);
#pragma unroll
        for (int i = 0; i < 4 * (D / 64); ++i) raw[i] = *(const u128 *)(J.q + at + 4 * i);
    }
    __device__ __forceinline__ void digest(const Job &J, int tile, unsigned long long *range) {
        const int col = threadIdx.x & 15;
        uint32_t l1 = 0, top = 0;                      // (l1: of a row that is not bad at most 32 x 2^23)
#pragma unroll
        for (int k = 0; k < D / 64; ++k) {
            uint32_t z[16];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const u128 v = raw[4 * k + i];
                const int32_t x[4] = {(int32_t)v.x, (int32_t)v.y, (int32_t)v.z, (int32_t)v.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t a = magnitude(x[j]);
                    l1 += a;
                    top = a > top ? a : top;
                    z[4 * i + j] = balanced(x[j]);
                }
            }
#pragma unroll
            for (int w = 0; w < 4; ++w) {              // four words' bytes to three digits' words
                uint32_t y[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) y[j] = z[channel_of(KB, 4 * w + j)];
                const uint32_t e = perm(y[1], y[0], 0x05010400u), f = perm(y[3], y[2], 0x05010400u);
                qd[0][k][w] = (int)perm(f, e, 0x05040100u);
                qd[1][k][w] = (int)perm(f, e, 0x07060302u);
                qd[2][k][w] = (int)perm(perm(y[3], y[2], 0x0C0C0602u), perm(y[1], y[0], 0x0C0C0602u), 0x05040100u);
            }
        }
        uint32_t out = 0;
        if (range && top >= (uint32_t)Q_ROT_LIMIT) {
#pragma unroll 1
            for (int i = 0; i < 4 * (D / 64); ++i) {
                const u128 v = *(const u128 *)(J.q + at + 4 * i);
                for (uint32_t x : {v.x, v.y, v.z, v.w}) out += magnitude((int32_t)x) >= (uint32_t)Q_ROT_LIMIT ? 1 : 0;
            }
        }
        double b1 = (double)l1 * J.kc_absmax;
        b1 += __shfl_xor(b1, 16);
        b1 += __shfl_xor(b1, 32);
        bad = row_or(top > 0x7F7F7Fu ? 1u : 0u) != 0 || !(b1 < DOT_MAX);
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

struct Digits {
    alignas(16) uint32_t dig[3][4];
    __device__ __forceinline__ void fill(int32_t c) {  // c: the thread's centroid, for 16 threads
        if (threadIdx.x < 16) {
            const uint32_t z = balanced(c);
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

// What a workgroup's tables are made of, a value a thread, requested together at its start.
struct Start {
    int32_t c, x;
    int parent;
    __device__ __forceinline__ Start(const Job &J, const Place &p, bool paths) {
        const int i = threadIdx.x;
        c = (int32_t)J.tabs->kc[i & 15];               // (no code names one behind the codebook's end)
        x = J.tabs->exp_table[i & 255];
        const int at = J.parents[p.b * J.pstride + imin(i, J.n - 1)];
        parent = paths && i < J.n ? at : -1;
    }
    // lut_s[floor(d log2(e) / 2^24)]: p by distance, the table an octave after the other (256 threads at least)
    __device__ __forceinline__ void lut(uint16_t *lut_s) const {
        if (threadIdx.x < 256) {
#pragma unroll
            for (int i = 0; i < LUT_SPAN / 256; ++i) lut_s[256 * i + threadIdx.x] = (uint16_t)(x >> i);
            if (threadIdx.x == 0) lut_s[LUT_SPAN] = 0;
        }
    }
};

// The value side: centroids / 2^23 and what follows from them.
template <int NC>
struct ValueTable {
    double vcs[NC], vcmax;
    uint32_t wide, delta_max;                          // wide: |v_norm p| up to which a term is two balanced bytes
    __device__ __forceinline__ explicit ValueTable(const Job &J) : vcmax(J.vcmax), wide(J.wide), delta_max(J.delta_max) {
#pragma unroll
        for (int i = 0; i < NC; ++i) vcs[i] = J.vcs[i];
    }
};

// RT row tiles a wave, which share the expanded keys.
template <int D, int KB, int RT>
__global__ void __launch_bounds__(W * 64, RT > 2 ? 3 : 4) max_kernel(Job J) {
    __shared__ Digits dgs;
    __shared__ uint32_t up[TREE_NODES][UPW];
    __shared__ int16_t at[TREE_NODES];
    Place p;
    if (!p.find(J, (J.tiles + RT - 1) / RT, J.mspan, W)) return;
    const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4, tile0 = p.tile * RT;
    const int nt = imin(RT, J.tiles - tile0);
    const Start start(J, p, p.tail);
    Query<D, KB> Q[RT];
    const uint32_t *path[RT];
    int32_t m[RT], lowest[RT];
    bool over[RT];
#pragma unroll
    for (int k = 0; k < RT; ++k) {
        const int tile = tile0 + imin(k, nt - 1);      // (a tile past the last one is not scored)
        Q[k].fetch(J, p, tile);
        path[k] = up[imin(tile * 16 + col, J.rows - 1) / J.g.G];
        m[k] = NONE;
        lowest[k] = 0;
    }
#pragma unroll
    for (int k = 0; k < RT; ++k) {
        Q[k].digest(J, tile0 + imin(k, nt - 1), J.count && p.s == 0 && k < nt ? &J.st->range_errors : nullptr);
        over[k] = Q[k].bad;
    }
    const uint8_t *hb = plane_ptr(J.g, p.b, p.kvh, 0), *nb = hb + (J.g.n_planes - 1) * J.g.span;
    Keys<D, KB> next;
    if (p.lo < p.hi) next.load(hb, nb, J.g.span, p.lo);
    dgs.fill(start.c);
    int none = 0;
    if (p.tail) none = tree_paths(start.parent, J.n, up, at);
    __syncthreads();
    if (J.count && none && p.kvh == 0 && p.tile == 0 && p.T <= (int64_t)(p.s / W + 1) * W * J.mspan)
        atomicAdd(&J.st->range_errors, (unsigned long long)none);
    if (p.lo >= p.hi) return;
    uint32_t dg[3][4];
    dgs.read(dg);
    for (int64_t t0 = p.lo; t0 < p.hi; t0 += 16) {
        const Keys<D, KB> cur = next;
        if (t0 + 16 < p.hi) next.load(hb, nb, J.g.span, t0 + 16);
        v4i a[D / 64][3];
        cur.expand(dg, a);
        const bool tail = t0 + 16 > p.base;
#pragma unroll
        for (int k = 0; k < RT; ++k) {
            if (k > 0 && k >= nt) break;
            uint32_t in = 15u;
            if (tail) in = visible4(path[k], (int)(t0 - p.base) + 4 * grp);
            int32_t s[4];
            over[k] |= scores<D>(a, Q[k].qd, cur.norms, Q[k].check, in, s);
            if (tail) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool on = in >> i & 1;
                    m[k] = on && s[i] > m[k] ? s[i] : m[k];
                    lowest[k] = on && s[i] < lowest[k] ? s[i] : lowest[k];
                }
            } else {
                m[k] = imax(m[k], imax(imax(s[0], s[1]), imax(s[2], s[3])));
                lowest[k] = imin(lowest[k], imin(imin(s[0], s[1]), imin(s[2], s[3])));
            }
        }
    }
#pragma unroll
    for (int k = 0; k < RT; ++k) {
        if (k >= nt) break;
        const int64_t tl = (int64_t)p.chain * J.tiles + tile0 + k, at0 = tl * J.nms + p.s;
        const int32_t top = row_max(m[k]);
        if (grp == 0) J.sc.top[at0 * 16 + col] = top;
        const uint64_t bad = __ballot(over[k]);
        if (lane == 0) {
            J.sc.over[at0] = (uint32_t)((bad | bad >> 16 | bad >> 32 | bad >> 48) & 0xFFFFu);
            if (p.s == 0) J.sc.pool[tl] = 0;
        }
        if (J.count) {
            const bool mine = !over[k] && (tile0 + k) * 16 + col < J.rows;
            const int64_t a = top == NONE ? 0 : top < 0 ? -(int64_t)top : top, c = -(int64_t)lowest[k];
            const int64_t x = wave_max_i64(mine ? (a > c ? a : c) : 0);
            if (lane == 0 && (unsigned long long)x > J.st->max_abs_score) atomicMax(&J.st->max_abs_score, (unsigned long long)x);
        }
    }
}

// A tile's value words, lane = tokens t0 + 4 grp .. + 3.
template <int D, int NC>
struct Values {
    static constexpr int VW = D * (NC == 8 ? 3 : 2) / 32;
    uint32_t w[4][VW];
    __device__ __forceinline__ void load(const uint8_t *vb0, int64_t span, int64_t t0, int vb) {
        const int64_t t = t0 + 4 * ((threadIdx.x & 63) >> 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (NC == 8 || vb == 2) {
#pragma unroll
                for (int p = 0; p < VW / 4; ++p) {
                    const uint4 v = *(const uint4 *)(vb0 + p * span + (t + i) * 16);
                    w[i][4 * p] = v.x;
                    w[i][4 * p + 1] = v.y;
                    w[i][4 * p + 2] = v.z;
                    w[i][4 * p + 3] = v.w;
                }
                if constexpr (VW % 4 != 0) {
                    const uint2 v = *(const uint2 *)(vb0 + (VW / 4) * span + (t + i) * 8);
                    w[i][VW - 2] = v.x;
                    w[i][VW - 1] = v.y;
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
    // the codes of channel 16 c + col, a byte a token
    __device__ __forceinline__ uint32_t codes(int c, int col) const {
        if constexpr (NC == 4) {
            const uint32_t b = (uint32_t)col >> 2, s = b | (4u + b) << 8;
            const uint32_t x = perm(w[1][c], w[0][c], s | 0x0C0C0000u) | perm(w[3][c], w[2][c], s << 16 | 0x0C0Cu);
            return x >> (2 * (col & 3)) & 0x03030303u;
        } else {
            // 16 channels are 48 bits, from bit 0 of word 3 c / 2 or bit 16 of the word before its end
            const int w0 = 48 * c / 32, sh = 48 * c % 32 + 3 * col;
            uint32_t x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t hi = w[i][w0 + 1], lo = sh < 32 ? w[i][w0] : hi;
                x[i] = __builtin_amdgcn_alignbit(hi, lo, sh & 31);
            }
            return (perm(x[1], x[0], 0x0C0C0400u) | perm(x[3], x[2], 0x04000C0Cu)) & 0x07070707u;
        }
    }
};

// 1 where a code (bytes of 4) is m.
__device__ __forceinline__ uint32_t is_code(int m, uint32_t codes) {
    return m < 4 ? perm(0u, 1u << (8 * m), codes) : perm(1u << (8 * (m - 4)), 0u, codes);
}

// A row tile's runs: 16 a span, the first of each row, and extra ones in order of demand. LDS: the first
// `near` of them in the workgroup's memory.
template <int D, bool LDS>
struct Runs {
    uint4 *meta, *meta_l;
    int32_t *S, *S_l;
    uint32_t *pool;
    int near;
    __device__ __forceinline__ Runs(const Job &J, const Place &p, uint4 *ml, int32_t *sl, int n, uint32_t *pl = nullptr)
        : meta_l(ml), S_l(sl), near(n) {
        const int64_t tl = (int64_t)p.chain * J.tiles + p.tile, run0 = tl * (16 * (int64_t)J.nspan + J.extra);
        meta = J.sc.meta + run0;
        S = J.sc.S + run0 * D;
        pool = LDS ? pl : J.sc.pool + tl;
    }
    // lane = (row, 4 channels of each 16), as the walk holds them
    __device__ __forceinline__ void put(int slot, const uint4 &m, const v4i (&acc)[D / 16], bool used) const {
        const int grp = (threadIdx.x & 63) >> 4;
        if (LDS && slot < near) {
            if (grp == 0) meta_l[slot] = m;
            if (!used) return;
#pragma unroll
            for (int c = 0; c < D / 16; ++c) *(v4i *)(S_l + slot * D + 16 * c + 4 * grp) = acc[c];
        } else {
            if (grp == 0) meta[slot] = m;
            if (!used) return;
#pragma unroll
            for (int c = 0; c < D / 16; ++c) *(v4i *)(S + (int64_t)slot * D + 16 * c + 4 * grp) = acc[c];
        }
    }
    __device__ __forceinline__ uint4 info(int slot) const { return LDS && slot < near ? meta_l[slot] : meta[slot]; }
    // of a wave-uniform run, lane = channel
    __device__ __forceinline__ void sum(int slot, bool used, int32_t (&v)[D / 64]) const {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int k = 0; k < D / 64; ++k)
            v[k] = !used ? 0 : LDS && slot < near ? S_l[slot * D + lane + 64 * k] : S[(int64_t)slot * D + lane + 64 * k];
    }
};

// A wave's walk over its span, from the maximum m before it (or, two-pass, of all): its runs into the
// scratch; returns the row's events, with BAD where it needs the serial path.
template <int D, int KB, int NC, bool LDS>
__device__ __forceinline__ uint32_t walk(const Job &J, const Place &p, const Query<D, KB> &Q, int32_t m,
                                         const ValueTable<NC> &values, const Runs<D, LDS> &runs, const Digits &dgs,
                                         const uint32_t *path, const uint16_t *lut_s) {
    constexpr int CT = D / 16, PVK = NC / 4;
    const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
    uint32_t dg[3][4];
    dgs.read(dg);
    const int vb = J.g.vb;
    const double (&vcs)[NC] = values.vcs, vcmax = values.vcmax;
    const uint32_t wide = values.wide, delta_max = values.delta_max;
    const uint8_t *hb = plane_ptr(J.g, p.b, p.kvh, 0), *nb = hb + (J.g.n_planes - 1) * J.g.span;
    const uint8_t *vb0 = hb + (int64_t)((J.g.key_bytes + 15) / 16) * J.g.span;
    bool first = p.s == 0;                             // what the span finds is nothing: it scales in place

    v4i acc[CT];                                       // lane = (row, 4 channels of each 16)
#pragma unroll
    for (int c = 0; c < CT; ++c) acc[c] = v4i{0, 0, 0, 0};
    uint32_t lp = 0;                                   // the lane's part of the denominator since the last event
    uint32_t l0 = 0;                                   // first span: the row's denominator up to there
    float bs = 0.0f;                                   // the lane's part of sum |v_norm p|
    const float bs_max = 0x1p28f / (float)fmax(vcmax, 0x1p-23);          // (four lanes: terms below 2^30, and a tile's)
    uint32_t wmax = 0;                                 // the largest |v_norm p|
    uint32_t n_ev = 0;                                 // the lane's events
    bool bad = Q.bad;
    int slot = p.s * 16 + col;                         // the row's open run (-1: none was left), and its factor
    uint32_t fopen = 1u << PROB_FRAC;

    auto lut = [&](uint32_t d) __attribute__((always_inline)) -> uint32_t {
        return lut_s[__umulhi(d, (uint32_t)LOG2E_Q16 << 8)];        // floor(d log2(e) / 2^24), d <= delta_max
    };
    auto clip = [&](int32_t hi, int32_t lo) __attribute__((always_inline)) -> uint32_t {
        const uint32_t w = (uint32_t)hi - (uint32_t)lo;
        return w < delta_max ? w : delta_max;
    };
    // the open run of the rows where `has`: into its record
    auto hand_over = [&](bool has, int next) __attribute__((always_inline)) {
        const uint32_t L = row_sum(lp);
        float b = bs;
        b += __shfl_xor(b, 16);
        b += __shfl_xor(b, 32);
        if (!has || slot < 0) return;
        const bool used = L != 0 || fopen != 1u << PROB_FRAC;
        const uint4 mt = make_uint4(L, fopen | (used ? USED : 0u), (uint32_t)next,
                                    __float_as_uint(b * (float)vcmax * 1.001f + (float)J.span));
        runs.put(slot, mt, acc, used);
    };
    // the run of the rows where `has` ends, and one with factor f begins. A row for which none is left goes token
    // by token and writes no more: every record is another row's, whose chain has to hold
    auto next_run = [&](bool has, uint32_t f) __attribute__((always_inline)) {
        int to = 0;
        if (has && grp == 0) to = (int)atomicAdd(runs.pool, 1u);
        to = __shfl(to, col);
        const bool none = to >= J.extra;
        bad = bad || (has && none);
        to = none ? -1 : 16 * J.nspan + to;
        hand_over(has, to);
        if (has) {
            slot = to;
            fopen = f;
            lp = 0;
            bs = 0.0f;
#pragma unroll
            for (int c = 0; c < CT; ++c) acc[c] = v4i{0, 0, 0, 0};
        }
    };

    Keys<D, KB> next;
    next.load(hb, nb, J.g.span, p.lo);
    for (int64_t t0 = p.lo; t0 < p.hi; t0 += 16) {
        const Keys<D, KB> cur = next;
        Values<D, NC> V;                               // (loaded before it is known whether any counts)
        V.load(vb0, J.g.span, t0, vb);
        if (t0 + 16 < p.hi) next.load(hb, nb, J.g.span, t0 + 16);
        const bool tail = t0 + 16 > p.base;
        int32_t s[4];
        uint32_t in = 15u;
        {
            v4i a[D / 64][3];
            cur.expand(dg, a);
            if (tail) in = visible4(path, (int)(t0 - p.base) + 4 * grp);
            scores<D>(a, Q.qd, cur.norms, false, in, s);
        }
        if (tail) {
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] = in >> i & 1 ? s[i] : NONE;
        }
        const int32_t mx = imax(imax(s[0], s[1]), imax(s[2], s[3]));
        const uint64_t evl = __ballot(mx > m);
        if (evl == 0 && __ballot((uint32_t)m - (uint32_t)mx < delta_max) == 0) continue;      // every p is 0
        const int32_t vn[4] = {(int32_t)cur.norms.x >> 16, (int32_t)cur.norms.y >> 16, (int32_t)cur.norms.z >> 16,
                               (int32_t)cur.norms.w >> 16};
        if (__ballot(bs > bs_max) != 0) {              // acc may leave 32 bits: it becomes a run
            first = false;
            lp += grp == 0 ? l0 : 0u;
            l0 = 0;
            next_run(true, 1u << PROB_FRAC);
        }
        uint32_t pw[4];
        const float bs0 = bs;
        v4i A[3][PVK];                     // the columns' digits
        auto weights = [&](const uint32_t (&dl)[4]) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < 4; ++i) pw[i] = lut(dl[i]);
            if (tail) {
#pragma unroll
                for (int i = 0; i < 4; ++i) pw[i] = in >> i & 1 ? pw[i] : 0u;
            }
        };
        // the terms for the weights; returns the largest |v_norm p|
        auto terms = [&](const uint32_t (&pp)[4]) __attribute__((always_inline)) -> uint32_t {
            uint32_t top = 0;
            double wd[4];
            uint32_t aw[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int32_t w = __mul24(vn[i], (int)pp[i]);
                aw[i] = w < 0 ? 0u - (uint32_t)w : (uint32_t)w;
                top = aw[i] > top ? aw[i] : top;
                bs += (float)aw[i];
                wd[i] = (double)w;
            }
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                uint32_t yl[4], yh[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint64_t y = (uint64_t)__double_as_longlong(fma(wd[i], vcs[c], TERM_MAGIC));
                    yl[i] = (uint32_t)y;
                    yh[i] = (uint32_t)(y >> 32);
                }
                const uint32_t l01 = perm(yl[1], yl[0], 0x0C0C0703u), l23 = perm(yl[3], yl[2], 0x07030C0Cu);
                const uint32_t h01 = perm(yh[1], yh[0], 0x05010400u), h23 = perm(yh[3], yh[2], 0x05010400u);
                A[0][c / 4][c % 4] = (int)((l01 | l23) ^ 0x80808080u);
                A[1][c / 4][c % 4] = (int)(perm(h23, h01, 0x05040100u) ^ 0x80808080u);
                A[2][c / 4][c % 4] = (int)(perm(h23, h01, 0x07060302u) ^ 0x80808080u);
            }
            return top;
        };
        // acc += the terms in A
        auto accumulate = [&](auto three, const v4i (&A)[3][PVK]) __attribute__((always_inline)) {
            // (opaque, so that the one-hot codes are made where they are used: kept over an events' loop they
            // take 32 registers and more, but for 16 where there are 4 codes and 4 tiles)
            int ch = col;
            if constexpr (CT * NC > 16) asm volatile("" : "+v"(ch));
            constexpr int GC = D == 64 ? 2 : 1;        // channel tiles at a time: registers
#pragma unroll
            for (int c0 = 0; c0 < CT; c0 += GC) {
                v4i oh[GC][PVK];
                v4i t[GC];
#pragma unroll
                for (int c = 0; c < GC; ++c) {
                    const uint32_t x = V.codes(c0 + c, ch);
#pragma unroll
                    for (int k = 0; k < NC; ++k) oh[c][k / 4][k % 4] = (int)is_code(k, x);
                    t[c] = v4i{0, 0, 0, 0};
                    if constexpr (decltype(three)::value) {
#pragma unroll
                        for (int k = 0; k < PVK; ++k) t[c] = mma(oh[c][k], A[2][k], t[c]);
                    }
                }
#pragma unroll
                for (int c = 0; c < GC; ++c) {
                    if constexpr (decltype(three)::value) t[c] = t[c] << 8;
#pragma unroll
                    for (int k = 0; k < PVK; ++k) t[c] = mma(oh[c][k], A[1][k], t[c]);
                }
#pragma unroll
                for (int c = 0; c < GC; ++c) {
                    t[c] = (t[c] << 8) + acc[c0 + c];
#pragma unroll
                    for (int k = 0; k < PVK; ++k) t[c] = mma(oh[c][k], A[0][k], t[c]);
                    acc[c0 + c] = t[c];
                }
            }
        };
        if (evl == 0) {
            const uint32_t dl[4] = {clip(m, s[0]), clip(m, s[1]), clip(m, s[2]), clip(m, s[3])};
            weights(dl);
            const uint32_t top = terms(pw);
            wmax = top > wmax ? top : wmax;
            lp += (pw[0] + pw[1]) + (pw[2] + pw[3]);
            if (__ballot(top > wide) == 0)
                accumulate(std::false_type{}, A);
            else
                accumulate(std::true_type{}, A);
            continue;
        }
        // events: the row's tokens fall into segments, one more than its events (bits 8 i of seg the segment of
        // token i)
        {
            int32_t e = m;                             // the maximum before the lane's tokens
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
                fe[i] = ev ? dd + 1u : 0u;             // an event's distance, + 1
                dl[i] = ev ? 0u : dd;
                e = ev ? s[i] : e;
                n += ev ? 1 : 0;
                seg |= n << (8 * i);
            }
            const uint32_t n1 = (uint32_t)__shfl((int)n, lane - 16), n2 = (uint32_t)__shfl((int)n, lane - 32),
                           n3 = (uint32_t)__shfl((int)n, lane - 48);
            const uint32_t off = (grp > 0 ? n1 : 0) + (grp > 1 ? n2 : 0) + (grp > 2 ? n3 : 0);
            seg += off * 0x01010101u;                  // at most 16
            const int row_ev = __shfl((int)(off + n), 48 + col);
            m = __shfl(e, 48 + col);
            n_ev += n;
            weights(dl);
            // a segment's terms are the tile's, masked, or made anew where the tile's would not fit beside them
            constexpr bool KEEP = CT * NC <= 16;
            uint32_t top = 0;
            if constexpr (KEEP) top = terms(pw);
            float bs_tile = bs - bs0;                  // (every run of the tile is bounded by all of it)
            for (int sg = 0;; ++sg) {
                uint32_t mask = 0, pp[4];              // the segment's tokens, a byte each
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool now = ((seg >> (8 * i)) & 0xFFu) == (uint32_t)sg;
                    mask |= now ? 0xFFu << (8 * i) : 0u;
                    pp[i] = now ? pw[i] : 0u;
                    lp += pp[i];
                }
                if constexpr (KEEP) {
                    v4i B[3][PVK];
#pragma unroll
                    for (int l = 0; l < 3; ++l)
#pragma unroll
                        for (int k = 0; k < PVK; ++k) B[l][k] = A[l][k] & (int)mask;
                    accumulate(std::true_type{}, B);
                } else {
                    top = terms(pp);
                    bs_tile = 0.0f;
                    accumulate(std::true_type{}, A);
                }
                wmax = top > wmax ? top : wmax;
                const bool has = row_ev > sg;
                if (__ballot(has) == 0) break;
                // the event that opens segment sg + 1 of the row
                uint32_t fd = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) fd = ((seg >> (8 * i)) & 0xFFu) == (uint32_t)(sg + 1) && fe[i] ? fe[i] : fd;
                fd = row_or(fd);
                const uint32_t f = has ? lut(fd - 1u) : 1u << PROB_FRAC;
                if (first) {
                    const uint32_t l = l0 + row_sum(lp);
                    if (has) {
#pragma unroll
                        for (int c = 0; c < CT; ++c) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                // floor(a f / 2^15) in halves of 16 bits: 2 hi f + floor(lo f / 2^15)
                                const uint32_t lo = __umul24((uint32_t)acc[c][i] & 0xFFFFu, f) >> PROB_FRAC;
                                acc[c][i] = __mul24(acc[c][i] >> 16, 2 * (int)f) + (int)lo;
                            }
                        }
                        l0 = (uint32_t)(((uint64_t)l * f) >> PROB_FRAC);
                        lp = 0;
                    }
                } else {
                    next_run(has, f);
                    bs = has ? bs_tile : bs;
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
    return events | any;
}

// Each row's largest of n spans' maxima (top: [span][16]), in the lanes of its column. A load takes 16 spans,
// lane = (span, 4 rows), and four of them are in flight: one by one a late span's hundred would cost more
// than its walk.
__device__ __forceinline__ int32_t top_of(const int32_t *top, int n) {
    const int lane = threadIdx.x & 63, col = lane & 15;
    int32_t m[4] = {NONE, NONE, NONE, NONE};
    for (int i0 = 0; i0 < n; i0 += 64) {
        int4 v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = i0 + 16 * j + (lane >> 2);
            v[j] = make_int4(NONE, NONE, NONE, NONE);
            if (i < n) v[j] = *(const int4 *)(top + (int64_t)i * 16 + 4 * (lane & 3));
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            m[0] = imax(m[0], v[j].x);
            m[1] = imax(m[1], v[j].y);
            m[2] = imax(m[2], v[j].z);
            m[3] = imax(m[3], v[j].w);
        }
    }
    int32_t mine = NONE;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
#pragma unroll
        for (int x = 4; x < 64; x *= 2) m[k] = imax(m[k], __shfl_xor(m[k], x));
        const int32_t y = __shfl(m[k], col >> 2);
        mine = (col & 3) == k ? y : mine;
    }
    return mine;
}

// OCC waves a SIMD.
template <int D, int KB, int NC, int OCC>
__global__ void __launch_bounds__(W * 64, OCC) sum_kernel(Job J) {
    __shared__ Digits dgs;
    __shared__ uint32_t up[TREE_NODES][UPW];
    __shared__ int16_t at[TREE_NODES];
    __shared__ uint16_t lut_s[LUT_N + 7];
    Place p;
    if (!p.find(J, J.tiles, J.span, W)) return;
    const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
    const Start start(J, p, p.tail);
    Query<D, KB> Q;
    Q.fetch(J, p, p.tile);
    // the maximum of the spans before, or of all
    int32_t m = NONE;
    if (p.lo < p.hi)
        m = top_of(J.sc.top + ((int64_t)p.chain * J.tiles + p.tile) * J.nms * 16,
                   J.two ? (int)((p.T + J.mspan - 1) / J.mspan) : p.s * (J.span / J.mspan));
    Q.digest(J, p.tile, nullptr);
    const ValueTable<NC> values(J);
    dgs.fill(start.c);
    start.lut(lut_s);
    if (p.tail) tree_paths(start.parent, J.n, up, at);
    __syncthreads();
    if (p.lo >= p.hi) return;
    const Runs<D, false> runs(J, p, nullptr, nullptr, 0);
    const uint32_t ev = walk<D, KB, NC, false>(J, p, Q, m, values, runs, dgs, up[imin(p.tile * 16 + col, J.rows - 1) / J.g.G], lut_s);
    if (grp == 0) J.sc.ev[(((int64_t)p.chain * J.tiles + p.tile) * J.nspan + p.s) * 16 + col] = ev;
}

// What a workgroup's rows count.
struct Tally {
    unsigned long long events, bad, over, acc, score;
    __device__ __forceinline__ void clear() { events = bad = over = acc = score = 0; }
    __device__ __forceinline__ void post(const Job &J, bool first, int64_t T) const {
        if (events) atomicAdd(&J.st->rescale_events, events);
        if (bad) atomicAdd(&J.st->serial_fallbacks, bad);
        if (over) atomicAdd(&J.st->acc_overflows, over);
        if (acc > J.st->max_abs_acc) atomicMax(&J.st->max_abs_acc, acc);
        if (score > J.st->max_abs_score) atomicMax(&J.st->max_abs_score, score);
        if (first) atomicMax(&J.st->n_tokens, (unsigned long long)T);
    }
};

// A wave puts row `col` of a tile together, lane = channel: its runs in order, then acc / l. False where the
// row has to go token by token.
template <int D, bool LDS>
__device__ __forceinline__ bool combine_row(const Job &J, const Place &p, int col, uint32_t events, const Runs<D, LDS> &runs,
                                            int32_t (*buf)[D], int32_t *list, Tally &tally) {
    constexpr int CPL = D / 64;
    const int lane = threadIdx.x & 63, r = p.tile * 16 + col, node = r / J.g.G;
    const int64_t qrow = (((int64_t)p.b * J.n + node) * J.g.n_q + p.kvh * J.g.G + r % J.g.G) * D;
    const int ns = (int)((p.T + J.span - 1) / J.span);
    int64_t acc[CPL];                                  // (online: what 32 bits hold)
    uint64_t l = 0;
#pragma unroll
    for (int k = 0; k < CPL; ++k) acc[k] = 0;
    bool bad = false;
    // one run after another; the loop is not unrolled, since its instructions come from memory but once
    auto apply = [&](uint32_t L, uint32_t f, float bound, const int32_t (&v)[CPL]) __attribute__((always_inline)) {
        if (J.two) {                                   // (no factors; clamped once, at the end)
#pragma unroll
            for (int k = 0; k < CPL; ++k) acc[k] += v[k];
            l += L;
            return;
        }
        const int32_t ff = (int32_t)(f & (USED - 1));
#pragma unroll
        for (int k = 0; k < CPL; ++k) {
            // floor(a f / 2^15) in halves of 16 bits, as in the walk
            const int32_t x = (int32_t)acc[k];
            const int32_t y = __mul24(x >> 16, 2 * ff) + (int32_t)(__umul24((uint32_t)x & 0xFFFFu, (uint32_t)ff) >> PROB_FRAC);
            bad = bad || !(fabsf((float)y) + bound <= 2147483000.0f);
            acc[k] = y + v[k];
        }
        l = ((l * (uint32_t)ff) >> PROB_FRAC) + L;
    };
    for (int i0 = 0; i0 < ns; i0 += 64) {
        const uint4 mt = i0 + lane < ns ? runs.info((i0 + lane) * 16 + col) : make_uint4(0u, 0u, ~0u, 0u);
        uint64_t todo = __ballot((mt.y & USED) != 0 || mt.z != ~0u);
        while (todo) {
            // (of the workgroup's memory they are read where they are; of the scratch, 16 at a time)
            uint64_t now = todo;
            if constexpr (!LDS) {
                constexpr int LR = D / 4, PER = 64 / LR;       // lanes a sum, 16 bytes each; sums a load
                const int rank = __popcll(todo & ((1ull << lane) - 1ull));
                wave_sync();
                if (todo >> lane & 1 && rank < 16) list[rank] = lane;
                now = __ballot((todo >> lane & 1) != 0 && rank < 16);
                wave_sync();
                const int cnt = __popcll(now);
                uint4 v[16 / PER];
#pragma unroll
                for (int j = 0; j < 16 / PER; ++j)
                    v[j] = *(const uint4 *)(runs.S + ((int64_t)(i0 + list[imin(PER * j + lane / LR, cnt - 1)]) * 16 + col) * D + 4 * (lane % LR));
#pragma unroll
                for (int j = 0; j < 16 / PER; ++j) *(uint4 *)&buf[PER * j + lane / LR][4 * (lane % LR)] = v[j];
                wave_sync();
            }
            todo &= ~now;
#pragma unroll 1
            for (int j = 0; now; ++j) {
                const int at = __ffsll((long long)now) - 1;
                now &= now - 1;
                uint32_t L = (uint32_t)__builtin_amdgcn_readlane((int)mt.x, at);
                uint32_t f = (uint32_t)__builtin_amdgcn_readlane((int)mt.y, at);
                int next = __builtin_amdgcn_readlane((int)mt.z, at);
                uint32_t bound = (uint32_t)__builtin_amdgcn_readlane((int)mt.w, at);
                int32_t v[CPL];
                if constexpr (LDS) {
                    runs.sum((i0 + at) * 16 + col, (f & USED) != 0, v);
                } else {
#pragma unroll
                    for (int k = 0; k < CPL; ++k) v[k] = buf[j][lane + 64 * k];
                }
#pragma unroll 1
                for (;;) {
                    if (f & USED) apply(L, f, __uint_as_float(bound), v);
                    if (next < 0) break;
                    const int slot = next;
                    const uint4 x = runs.info(slot);
                    L = (uint32_t)uni32((int)x.x);
                    f = (uint32_t)uni32((int)x.y);
                    next = uni32((int)x.z);
                    bound = (uint32_t)uni32((int)x.w);
                    runs.sum(slot, (f & USED) != 0, v);
                }
            }
        }
    }
    if (__ballot(bad) != 0) return false;
    const Recip rc = reciprocal((int64_t)l);
    int64_t amax = 0, over = 0;
#pragma unroll
    for (int k = 0; k < CPL; ++k) {
        if (acc[k] < ACC_LO || acc[k] > ACC_HI) {
            ++over;
            acc[k] = acc[k] < ACC_LO ? ACC_LO : ACC_HI;
        }
        J.out[qrow + lane + 64 * k] = (int32_t)(wmul(acc[k], rc.r) >> rc.shift);
        const int64_t m = acc[k] < 0 ? -acc[k] : acc[k];
        amax = m > amax ? m : amax;
    }
    if (J.count) {
        const int64_t ev = wave_sum_i64((int64_t)events);
        amax = wave_max_i64(amax);
        over = wave_sum_i64(over);
        if (lane == 0) {
            if (ev && !J.two) atomicAdd(&tally.events, (unsigned long long)ev);
            if (over) atomicAdd(&tally.over, (unsigned long long)over);
            atomicMax(&tally.acc, (unsigned long long)amax);
        }
    }
    return true;
}

template <int D>
using RowLds = SerialLds<D == 64 ? 60 : 116>;          // (the widest row: 4-bit keys, 3-bit values)
template <int D>
__device__ __forceinline__ void serial_row(const Job &J, const Place &p, int col, RowLds<D> &fb, uint32_t *up, Tally &tally) {
    const int r = p.tile * 16 + col, node = r / J.g.G;
    const int64_t qrow = (((int64_t)p.b * J.n + node) * J.g.n_q + p.kvh * J.g.G + r % J.g.G) * D;
    tree_path(J.parents + p.b * J.pstride, node, J.n, up);
    serial_head<D / 64, (D == 64 ? 60 : 116)>(J.g, J.tabs, J.tabs->kc, J.tabs->vc, J.q + qrow, p.b, p.kvh, p.T, J.two, true, fb,
                                              J.out + qrow, J.st, TreeRows{up, p.base});
    if ((threadIdx.x & 63) == 0) atomicAdd(&tally.bad, 1ull);
}

template <int D>
__global__ void __launch_bounds__(CW * 64) combine_kernel(Job J) {
    __shared__ union {
        RowLds<D> fb;
        alignas(16) int32_t buf[16][D];
    } u[CW];
    __shared__ int32_t list[CW][16];
    __shared__ uint32_t up[CW][TREE_NODES / 32];
    __shared__ Tally tally;
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int chains = J.nseq * J.g.n_kv;
    const int part = (int)(blockIdx.x / (unsigned)chains);
    Place p;
    p.chain = (int)(blockIdx.x % (unsigned)chains);
    p.tile = part / (16 / CW);
    p.b = J.seq0 + p.chain / J.g.n_kv;
    p.kvh = p.chain % J.g.n_kv;
    p.T = rows_of(J, p.b);
    p.base = p.T - J.n;
    if (tid == 0) tally.clear();
    __syncthreads();
    const int col = part % (16 / CW) * CW + wv;
    if (p.tile * 16 + col < J.rows) {
        const int64_t tl = (int64_t)p.chain * J.tiles + p.tile;
        const int ns = (int)((p.T + J.span - 1) / J.span), nm = (int)((p.T + J.mspan - 1) / J.mspan);
        uint32_t events = 0;
        bool bad = false;
        for (int i = lane; i < ns; i += 64) {
            const uint32_t e = J.sc.ev[(tl * J.nspan + i) * 16 + col];
            events += e & ~BAD;
            bad = bad || (e & BAD) != 0;
        }
        for (int i = lane; i < nm; i += 64) bad = bad || (J.sc.over[tl * J.nms + i] >> col & 1) != 0;
        const Runs<D, false> runs(J, p, nullptr, nullptr, 0);
        if (__ballot(bad) != 0 || !combine_row<D, false>(J, p, col, events, runs, u[wv].buf, list[wv], tally))
            serial_row<D>(J, p, col, u[wv].fb, up[wv], tally);
    }
    if (!J.count) return;
    __syncthreads();
    if (tid == 0) tally.post(J, part == 0 && p.kvh == 0, p.T);
}

// All of it in one launch, where the spans are a workgroup's waves (19 us for 5 nodes behind 100 tokens, a chain of
// waits: tables and queries 4, maxima 1, walk 6, runs 5; the rest launch and end).
constexpr int FW = 8;
template <int D, int KB, int NC>
__global__ void __launch_bounds__(FW * 64, 2) fused_kernel(Job J) {
    __shared__ Digits dgs;
    __shared__ uint32_t up[TREE_NODES][UPW];
    __shared__ int16_t at[TREE_NODES];
    __shared__ uint16_t lut_s[LUT_N + 7];
    __shared__ int32_t top_s[FW][16];
    __shared__ uint32_t bad_s, pool_s, ev_s[FW][16];
    __shared__ Tally tally;
    constexpr int NEAR = D == 64 ? 192 : 160;
    __shared__ union {
        struct {
            uint4 meta[NEAR];
            int32_t S[NEAR][D];
        } r;
        struct {
            RowLds<D> fb[FW];
            uint32_t up[FW][TREE_NODES / 32];
        } f;
    } u;
    Place p;
    p.find(J, J.tiles, J.span, FW);
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, grp = lane >> 4;
    Query<D, KB> Q;
    Q.fetch(J, p, p.tile);
    const Start start(J, p, true);
    const uint8_t *hb = plane_ptr(J.g, p.b, p.kvh, 0), *nb = hb + (J.g.n_planes - 1) * J.g.span;
    Keys<D, KB> next;
    if (p.lo < p.hi) next.load(hb, nb, J.g.span, p.lo);
    const ValueTable<NC> values(J);
    Q.digest(J, p.tile, J.count && p.s == 0 ? &J.st->range_errors : nullptr);
    const Runs<D, true> runs(J, p, u.r.meta, u.r.S[0], NEAR, &pool_s);
    dgs.fill(start.c);
    start.lut(lut_s);
    if (tid == 0) {
        bad_s = 0;
        tally.clear();
        pool_s = 0;
    }
    const int none = tree_paths(start.parent, J.n, up, at);
    if (J.count && none && p.kvh == 0 && p.tile == 0) atomicAdd(&J.st->range_errors, (unsigned long long)none);
    __syncthreads();
    const uint32_t *path = up[imin(p.tile * 16 + col, J.rows - 1) / J.g.G];
    int32_t m = NONE;
    if (p.lo < p.hi) {
        int32_t lowest = 0;
        bool over = Q.bad;
        uint32_t dg[3][4];
        dgs.read(dg);
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
        m = row_max(m);
        const uint64_t bad = __ballot(over);
        if (lane == 0 && bad) atomicOr(&bad_s, (uint32_t)((bad | bad >> 16 | bad >> 32 | bad >> 48) & 0xFFFFu));
        if (J.count) {
            const bool mine = !over && p.tile * 16 + col < J.rows;
            const int64_t x = m == NONE ? 0 : m < 0 ? -(int64_t)m : m, y = -(int64_t)lowest;
            const int64_t z = wave_max_i64(mine ? (x > y ? x : y) : 0);
            if (lane == 0) atomicMax(&tally.score, (unsigned long long)z);
        }
    }
    if (grp == 0) top_s[p.s][col] = m;
    __syncthreads();
    if (p.lo < p.hi) {
        m = NONE;
        for (int i = 0; i < (J.two ? FW : p.s); ++i) m = imax(m, top_s[i][col]);
        const uint32_t ev = walk<D, KB, NC, true>(J, p, Q, m, values, runs, dgs, path, lut_s);
        if (grp == 0) ev_s[p.s][col] = ev;
    } else if (grp == 0) {
        ev_s[p.s][col] = 0;
    }
    __syncthreads();
    for (int c = p.s; c < 16; c += FW) {
        if (p.tile * 16 + c >= J.rows) break;
        const uint32_t e = lane < FW ? ev_s[lane][c] : 0u;
        const bool bad = __ballot((e & BAD) != 0) != 0 || (bad_s >> c & 1) != 0;
        if (bad || !combine_row<D, true>(J, p, c, e & ~BAD, runs, nullptr, nullptr, tally)) {
            if (lane == 0) atomicOr(&bad_s, 1u << (16 + c));
        }
    }
    __syncthreads();                                   // (the serial path's rows lie over the runs)
    const uint32_t bad = (uint32_t)uni32((int)(bad_s >> 16));
    for (int c = p.s; c < 16; c += FW)
        if (bad >> c & 1) serial_row<D>(J, p, c, u.f.fb[p.s], u.f.up[p.s], tally);
    if (!J.count) return;
    __syncthreads();
    if (tid == 0) tally.post(J, p.tile == 0 && p.kvh == 0, p.T);
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
    const int64_t T = rows_of(J, b);
    serial_head<CPL, SERIAL_RS>(J.g, J.tabs, kc, vc, J.q + at, b, qh / J.g.G, T, J.two, true, L, J.out + at, J.st,
                                TreeRows{up, T - J.n});
}

namespace {
// Sequences a launch takes, and the spans of the longest.
struct Plan {
    int64_t seqs, tiles, span, nspan, mspan, nms, rt, extra;
    bool fused, longw;
};
// The scratch of a launch, carved from p (null: only its size).
size_t carve(const Geom &g, const Plan &pl, uint8_t *p, Scratch *sc) {
    const int64_t nseq = pl.seqs, tiles = pl.tiles, nspan = pl.nspan, nms = pl.nms;
    size_t o = 0;
    auto take = [&](size_t n) {
        uint8_t *a = p ? p + o : nullptr;
        o += (n + 255) / 256 * 256;
        return a;
    };
    const size_t all = (size_t)nseq * g.n_kv * tiles, runs = all * (16 * (size_t)nspan + pl.extra);
    Scratch c{};
    c.top = (int32_t *)take(all * nms * 64);
    c.over = (uint32_t *)take(all * nms * 4);
    c.ev = (uint32_t *)take(all * nspan * 64);
    c.pool = (uint32_t *)take(all * 4);
    c.meta = (uint4 *)take(runs * 16);
    c.S = (int32_t *)take(runs * g.d * 4);
    if (sc) *sc = c;
    return o;
}

constexpr size_t BUDGET = (size_t)512 << 20;
// Contexts up to here in one launch (4b/2b, 32 heads of 64 over 8, online, call to call: 5 nodes behind 100 tokens 18.6
// us, in three launches 27.0; 26 behind 486: 29.2 and 30.4; behind 1,000: 42.6 and 33.8; 26 x 8 sequences behind 100,
// 486 and 1,000: 35.7 and 36.8, 55.6 and 53.0, 82.0 and 84.9). Of many row tiles three would be the faster way at any
// length, since its registers leave a CU one workgroup: 64 nodes x 8 sequences behind 100: 77.7 and 59.8, x 32: 298 and
// 169; 256 x 8: 389 and 225.
constexpr int64_t FUSED_MAX = 512;
Plan plan(const Geom &g, int64_t n, int64_t longest, int64_t batch) {
    Plan p{};
    p.tiles = (n * g.G + 15) / 16;
    p.seqs = batch;
    for (;;) {
        const int64_t all = p.seqs * g.n_kv * p.tiles;
        // row tiles a wave of max_kernel: as many as leave it 4,096 waves of 64 tokens (64 nodes behind 4,097 tokens:
        // two 57 us, four 61; 26 behind 8,192 x 8 sequences: four 193, two 200; 9 x 16 ragged: four 147, one 164)
        p.rt = g.d == 64 ? 4 : 2;
        while (p.rt > 1 && (p.tiles <= p.rt / 2 || p.seqs * g.n_kv * ((p.tiles + p.rt - 1) / p.rt) * ((longest + 63) / 64) < 4096)) p.rt /= 2;
        const int64_t most = (longest + 63) / 64, least = (longest + SPAN_MAX - 1) / SPAN_MAX;
        // spans: as many waves of sum_kernel as the chip holds at two a SIMD. Where they would walk more than 300 tokens
        // each: with 4 value codes at d = 64 three a SIMD, for which some registers go to memory (13 nodes x 4 behind
        // 2,047 tokens: two a SIMD 58 us, three 62; 26 behind 32,768: 120 and 110), and up to three rounds of them
        // while that leaves 256 tokens, since later ones even out ragged ends and first spans' events (9 nodes x 16
        // ragged: one 177, two 147, three 140; 5 x 3 behind 20,000, 105 tokens each in three: one 95, three 109)
        int64_t want = 2048 / all;
        p.longw = longest > 300 * want;
        if (p.longw) {
            const int64_t round = std::max<int64_t>(1024 * (g.d == 64 && g.vb <= 2 ? 3 : 2) / all, 1);
            want = round * std::min<int64_t>(std::max<int64_t>(longest / (256 * round), 1), 3);
        }
        want = std::max<int64_t>(std::min(want, most), std::max<int64_t>(least, 1));
        p.fused = longest <= FUSED_MAX;
        if (p.fused) {
            p.span = ((longest + FW - 1) / FW + 15) / 16 * 16;
            p.nspan = FW;
        } else {
            // a multiple of 64 tokens, so that up to four of max_kernel's make one
            p.span = ((longest + want - 1) / want + 63) / 64 * 64;
            p.nspan = (longest + p.span - 1) / p.span;
        }
        // max_kernel's waves: a round of them where each still walks 128 tokens, half a round else: what comes
        // before a walk costs as much as some 50 tokens (26 nodes behind 32,768: 160 tokens a wave 42 us, 80 tokens
        // 44; 9 nodes x 16 ragged sequences: 144 tokens 46 us, 288 tokens 50)
        p.mspan = p.span;
        auto waves = [&] { return p.seqs * g.n_kv * ((p.tiles + p.rt - 1) / p.rt) * ((longest + p.mspan - 1) / p.mspan); };
        while (!p.fused && p.mspan % 32 == 0 && p.span / p.mspan < 4 && waves() < (p.mspan >= 256 ? 4096 : 2048)) p.mspan /= 2;
        p.nms = (longest + p.mspan - 1) / p.mspan;
        const int64_t room = (64 << 20) / (all * (g.d * 4 + 16));
        p.extra = room < EXTRA_MIN ? EXTRA_MIN : room > EXTRA_MAX ? EXTRA_MAX : room;
        if (p.seqs == 1 || carve(g, p, nullptr, nullptr) <= BUDGET) return p;
        p.seqs = (p.seqs + 1) / 2;
    }
}

}  // namespace

template <int D, int KB, int NC>
hipError_t launch(hipStream_t s, const Job &J, int rt, bool fused, bool longw, LaunchEv ev) {
    const int64_t chains = (int64_t)J.nseq * J.g.n_kv;
    if (fused) {
        hipExtLaunchKernelGGL((fused_kernel<D, KB, NC>), dim3((unsigned)(chains * J.tiles)), dim3(FW * 64), 0, s, ev.start, ev.stop, 0, J);
        return hipGetLastError();
    }
    const dim3 grid((unsigned)(chains * J.tiles * ((J.nspan + W - 1) / W)));
    const int64_t ms = (J.nms + W - 1) / W;
    if (rt == 1)
        hipExtLaunchKernelGGL((max_kernel<D, KB, 1>), dim3((unsigned)(chains * ms * J.tiles)), dim3(W * 64), 0, s, ev.start, nullptr, 0, J);
    else if (D == 128 || rt == 2)
        hipExtLaunchKernelGGL((max_kernel<D, KB, 2>), dim3((unsigned)(chains * ms * ((J.tiles + 1) / 2))), dim3(W * 64), 0, s, ev.start, nullptr, 0, J);
    else
        hipExtLaunchKernelGGL((max_kernel<D, KB, D == 128 ? 2 : 4>), dim3((unsigned)(chains * ms * ((J.tiles + 3) / 4))), dim3(W * 64), 0, s, ev.start, nullptr, 0, J);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    constexpr int OCC = D == 64 && NC == 4 ? 3 : 2;
    if (longw)
        hipExtLaunchKernelGGL((sum_kernel<D, KB, NC, OCC>), grid, dim3(W * 64), 0, s, nullptr, nullptr, 0, J);
    else
        hipExtLaunchKernelGGL((sum_kernel<D, KB, NC, 2>), grid, dim3(W * 64), 0, s, nullptr, nullptr, 0, J);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipExtLaunchKernelGGL((combine_kernel<D>), dim3((unsigned)(chains * ((J.rows + CW - 1) / CW))), dim3(CW * 64), 0, s, nullptr, ev.stop, 0, J);
    return hipGetLastError();
}

}  // namespace tr

bool tree_supported(const Geom &g) {
    return (g.d == 64 || g.d == 128) && g.kb >= 2 && g.kb <= 4 && g.vb >= 1 && g.vb <= 3 && g.norm_frac == 9;
}

size_t tree_scratch_bytes(const Geom &g, int64_t n, int64_t longest) {
    const tr::Plan p = tr::plan(g, n, longest, g.batch);
    return tr::carve(g, p, nullptr, nullptr);
}

hipError_t launch_attend_tree(hipStream_t s, const Geom &g, const Tables *t, const Tables &host, const int32_t *q, int32_t *out,
                              const int64_t *len, const int32_t *parents, int64_t pstride, int32_t n, int64_t longest,
                              int two_pass, bool count, void *scratch, size_t scratch_bytes, LaunchEv ev, DevStats *st) {
    using namespace tr;
    const Plan p = plan(g, n, longest, g.batch);
    Job J{};
    if (carve(g, p, (uint8_t *)scratch, &J.sc) > scratch_bytes) return hipErrorInvalidValue;
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
    J.mspan = (int32_t)p.mspan;
    J.nms = (int32_t)p.nms;
    J.extra = (int32_t)p.extra;
    J.two = two_pass;
    J.count = count;
    J.longest = longest;
    J.kc_absmax = host.kc_absmax;
    for (int i = 0; i < 1 << g.vb; ++i) {
        J.vcs[i] = (double)host.vc[i] * 0x1p-23;
        J.vcmax = std::fmax(J.vcmax, std::fabs(J.vcs[i]));
    }
    J.wide = (uint32_t)(32639.0 / std::fmax(J.vcmax, 0x1p-16));
    J.delta_max = (uint32_t)host.delta_max;
    J.st = st;
    for (int64_t b = 0; b < g.batch; b += p.seqs) {
        J.seq0 = (int32_t)b;
        J.nseq = (int32_t)std::min<int64_t>(p.seqs, g.batch - b);
        const LaunchEv e{b == 0 ? ev.start : nullptr, b + p.seqs >= g.batch ? ev.stop : nullptr};
        hipError_t rc = hipErrorInvalidValue;
#define INSITU_TREE_CASE(DD, KK, CC) \
    if (g.d == DD && g.kb == KK && (g.vb <= 2 ? 4 : 8) == CC) rc = launch<DD, KK, CC>(s, J, (int)p.rt, p.fused, p.longw, e);
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
                                     const int64_t *len, const int32_t *parents, int64_t pstride, int32_t n, int64_t longest,
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
    J.longest = longest;
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
