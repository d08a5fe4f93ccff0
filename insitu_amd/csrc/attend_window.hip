// The attend of layers with a sliding window (and a few first rows that stay visible): the last n rows of a
// sequence are the queries' own, and the query at row p attends, in row order, the rows t <= p with t < sinks
// or t > p - window, with the integers that attend_online / attend_two_pass (ops/attention.py:429-513) give
// on those rows. The reference attends all of a context and has no counterpart.
//
// Many queries run on the prefill kernel (attend_prefill.hip), a wave 16 (query, head) rows over all they see.
// Here are the few of decode steps and short turns (span_kernel), which leave the chip to so few such waves that
// the walk of one is the time: a workgroup holds one tile of R rows, 4, 8 or 16, of a KV head, and its eight or
// twelve waves share out what the tile sees, in order; behind barriers follow
//   the scores     of each wave's span, kept in LDS, and their largest a row;
//   the walk       with the maximum of the spans before (online) or of all (two-pass). The terms
//                  floor(v_norm p c / 2^23) between two rises of the maximum (events) are only added: such a run
//                  gives a sum S and a denominator L without knowing what came before, and the factor f that its
//                  event scales that by. The first span, which begins with nothing, scales in place;
//   the runs       acc = floor(acc f / 2^15) + S, l = floor(l f / 2^15) + L in order, the recurrence itself as
//                  long as the clamp of acc after every token cannot fire, which |acc| plus the sum of a run's
//                  |terms| below 2^31 proves. Then acc / l.
// A row that cannot be proven (also: a query value past three digits, a score past 32 bits, a term past three
// digits, more runs than there is room for) is recomputed token by token (serial_head.h).
//
// Matrix operands as in the prefill kernel: three balanced digits of q and of the centroids for the scores, three
// of the terms times one-hot value codes for the sums. A product's 16 columns are R rows times J = 16 / R groups of
// 16 tokens: the query digits of the other groups' columns are zero, so that J products into one accumulator
// leave every lane a score of its own, and one lane's arithmetic (scores, weights, terms) serves one row and
// 4 of the step's 16 J tokens; for one token's four query heads a quarter of what 16 rows a tile would take.
// The terms' digits are summed apart and put together where a run ends. A lane's channels lie together in the
// value codes (channel col D / 16 + c in product c), so that it reads a word of a row, not all of it.
//
// What bounds it: VALU issue, and in a small call the chain of one workgroup's phases. A decode token of 32 sequences
// of 8 KV heads over 4,096 rows (53.7 us; 11.8 to read them at the rate of a copy) is a workgroup a CU and three waves a
// SIMD, which issue VALU 60 % of the time: tables and queries 3 us, keys expanded and scores 16, the walk 22 (10 of it
// events: two-pass, which has none, takes 43), the runs 2. A wave a (token, head), token by token, takes 1,807 us; the
// prefill kernel, whose workgroup's 64 rows are 4 here, 326. One query over a window of 128 in 300 rows, 15.8 us with the
// call, is mostly instructions that come from memory once: loops that are not unrolled are faster there. At d = 128, or
// with 8 codes a value, eight waves: twelve have too few registers.
// A tile's window stays on one CU however long it is, so that one sequence's token takes as long as that of 32 (52 us of
// 4,096 rows, on 8 CUs) and longer than all of a long context, which the dense attends spread over the chip (16,384 rows
// 177 us, 32,768 rows there 66). Nothing in the integers asks for that, two-pass least of all, whose sums have no order.
#include <algorithm>
#include <cmath>

#include "digits.h"
#include "query.h"
#include "row_codec.h"
#include "serial_head.h"
#include "wave.h"

namespace insitu {
namespace wn {

// The row behind query i's own of sequence b, and what it sees.
__device__ __forceinline__ int64_t end_of(const WindowJob &w, int b, int64_t i) {
    const int64_t T = w.len[b] > w.n ? w.len[b] : w.n;
    return T - w.n + i + 1;
}
__device__ __forceinline__ WindowRows rows_of(const WindowJob &w, int64_t end) {
    return WindowRows{w.sinks, end > w.window ? end - w.window : 0};
}

constexpr float EVENTS = 8.0f, EVENTS_FROM = 5.0f;     // of span_start, in tiles
constexpr int DPP_ROW_ROR4 = 0x124, DPP_ROW_ROR12 = 0x12C;       // lane i <- lane (i - 4), (i + 4) mod 16 of its row
constexpr int RUN_MAX = 32768;                         // tokens of a run, so that its L fits 32 bits
constexpr uint32_t LUT_N = LUT_SPAN + 1;
constexpr double TERM_MAGIC = 402653184.0 + 8421504.0; // 1.5 * 2^28 + 0x808080: ulp 2^-24
constexpr double TERM_LIMIT = 8355711.0;               // 0x7F7F7F: three balanced bytes
constexpr double DOT_MAX = 0x1p46;                     // ||q||_1 max|c| below it: dot / 2^16 fits int32
constexpr double NARROW_LIMIT = 36028797018963968.0 - 16777216.0;   // |dot k_norm| below it: the score fits int32
constexpr int32_t NONE = INT32_MIN;                    // no score
constexpr uint32_t BAD = 1u << 31, USED = 1u << 16;

struct __attribute__((aligned(4))) u128 {              // 16 bytes of a 4-byte aligned address
    uint32_t x, y, z, w;
};

struct Job {
    Geom g;
    const Tables *tabs;
    WindowJob w;
    int32_t rows;                                      // n G, of a (sequence, KV head)
    uint32_t first;                                    // the launch's first workgroup of all
    int32_t chains, extra, count;                      // extra: runs a workgroup has in the scratch; count: statistics
    double kc_absmax, vcs[8], vcmax;                   // vcs: value centroids / 2^23
    uint32_t wide, delta_max;                          // wide: |v_norm p| up to which a term is two balanced bytes
    uint4 *meta;                                       // [workgroup][run]: L, f | USED, the span's next run or -1, a bound (float)
    int32_t *S;                                        // [workgroup][run][d]
    DevStats *st;
};

__device__ __forceinline__ int32_t imax(int32_t a, int32_t b) { return a > b ? a : b; }
__device__ __forceinline__ int32_t imin(int32_t a, int32_t b) { return a < b ? a : b; }
__device__ __forceinline__ uint32_t magnitude(int32_t x) { return x < 0 ? 0u - (uint32_t)x : (uint32_t)x; }

// A barrier for what LDS holds: loads and stores of memory stay in flight.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}
// The value of the lane R j columns on, in turn: tokens' group j in the place of the first.
template <int R>
__device__ __forceinline__ uint32_t group_of(int j, uint32_t v) {
    if constexpr (R == 16) return v;
    // (every lane has a source; the compiler then takes the move into the instruction that uses it)
    if (j == 0) return v;
    if (R == 8 || j == 2) return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, DPP_ROW_ROR8, 0xF, 0xF, true);
    if (j == 1) return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, DPP_ROW_ROR12, 0xF, 0xF, true);
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, DPP_ROW_ROR4, 0xF, 0xF, true);
}
// Over the lanes of a row: its column of every group of tokens (R apart), four times 16 lanes.
template <int R, class F>
__device__ __forceinline__ uint32_t row_all(uint32_t v, F f) {
    const int lane = threadIdx.x & 63;
    if constexpr (R <= 4) v = f(v, xor_lane32<4>(v, lane));
    if constexpr (R <= 8) v = f(v, xor_lane32<8>(v, lane));
    v = f(v, xor_lane32<16>(v, lane));
    return f(v, xor_lane32<32>(v, lane));
}
template <int R>
__device__ __forceinline__ int32_t row_max(int32_t v) {
    return (int32_t)row_all<R>((uint32_t)v, [](uint32_t a, uint32_t b) { return (uint32_t)imax((int32_t)a, (int32_t)b); });
}
template <int R>
__device__ __forceinline__ uint32_t row_or(uint32_t v) {
    return row_all<R>(v, [](uint32_t a, uint32_t b) { return a | b; });
}
template <int R>
__device__ __forceinline__ uint32_t row_sum(uint32_t v) {
    return row_all<R>(v, [](uint32_t a, uint32_t b) { return a + b; });
}

// Lane i <= FW: the tile that span i of FW begins with (of nt; span FW is the end). Events thin out as 1 / x along what
// a tile of rows sees, so that its first x tiles take about x + a ln(1 + x / EVENTS_FROM) times a tile without any: the
// spans share that out evenly (Newton; its start is behind the cut, and the steps after the first stay before it). Equal
// spans take 62 us where these take 55 (a decode token of 32 sequences, window 4,096), 38.8 where 37 (16 tokens, 1,024).
template <int FW>
__device__ __forceinline__ int span_start(int nt, float a) {
    const int i = threadIdx.x & 63;
    if (nt <= FW) return imin(i, nt);
    const float rate = 1.0f / EVENTS_FROM, al = a * 0.693147181f, n = (float)nt;
    const float goal = (n + al * __builtin_amdgcn_logf(1.0f + n * rate)) * ((float)i / FW);
    float x = n * ((float)i / FW);
#pragma unroll 1
    for (int k = 0; k < 4; ++k) {
        const float y = 1.0f + x * rate, c = x + al * __builtin_amdgcn_logf(y);
        x = fmaxf(x + (goal - c) * __builtin_amdgcn_rcpf(1.0f + a * rate * __builtin_amdgcn_rcpf(y)), 0.0f);
    }
    const int t = (int)(x + 0.5f);
    return i <= 0 ? 0 : i >= FW ? nt : imin(imax(t, 1), nt);
}

// A workgroup's tile of rows and the rows of the cache that it sees: the 16-row tiles of the first rows and those
// from the first row's window on, U rows numbered on end.
template <int R>
struct Place {
    int b, seq, kvh;                                   // sequence of the call, of the cache
    int row0;                                          // the tile's first row
    int64_t len;                                       // (requested first, used last)
    int64_t base, U;                                   // the first query's own row; what the tile sees
    int64_t skip_at, skip;                             // where numbers and rows part, and how far
    int64_t first_end, last_lo;                        // the first row's end, where the last row's window begins
    __device__ __forceinline__ explicit Place(const Job &J) {
        const uint32_t wg = J.first + blockIdx.x, chain = wg % (uint32_t)J.chains;
        row0 = (int)(wg / (uint32_t)J.chains) * R;
        b = (int)(chain / (uint32_t)J.g.n_kv);
        kvh = (int)(chain % (uint32_t)J.g.n_kv);
        seq = J.w.seq_lo + b;
        len = J.w.len[seq];
    }
    __device__ __forceinline__ void find(const Job &J) {
        base = (len > J.w.n ? len : J.w.n) - J.w.n;
        const int last = (row0 + R < J.rows ? row0 + R : J.rows) - 1;
        first_end = base + (uint32_t)row0 / (uint32_t)J.g.G + 1;
        const int64_t end = base + (uint32_t)last / (uint32_t)J.g.G + 1, lo = first_end - J.w.window;
        last_lo = end - J.w.window;
        skip_at = (J.w.sinks + 15) & ~(int64_t)15;
        skip = lo > skip_at ? (lo & ~(int64_t)15) - skip_at : 0;
        U = end - skip;
    }
    __device__ __forceinline__ int64_t at(int64_t u) const { return u < skip_at ? u : u + skip; }      // u a multiple of 16
    // of row r of the KV head: its query's place among the queries, and its own row's end
    __device__ __forceinline__ int64_t query(const Job &J, int r) const {
        const uint32_t G = (uint32_t)J.g.G, i = (uint32_t)r / G;
        return ((int64_t)b * J.w.n + i) * J.g.n_q + kvh * G + ((uint32_t)r - i * G);
    }
    __device__ __forceinline__ int64_t end(const Job &J, int r) const { return base + (uint32_t)r / (uint32_t)J.g.G + 1; }
};

// A row's queries, lane = (row, D / 4 channels from grp D / 4 on, in the order the codes expand in), as digits.
template <int D, int KB>
struct Query {
    v4i qd[3][D / 64];
    bool bad, check;                                   // needs the serial path; scores may leave int32
    uint32_t out;                                      // values out of range
    u128 raw[4 * (D / 64)];
    __device__ __forceinline__ void fetch(const int32_t *q) {
#pragma unroll
        for (int i = 0; i < 4 * (D / 64); ++i) raw[i] = *(const u128 *)(q + 4 * i);
    }
    __device__ __forceinline__ void make(double kc_absmax) {
        uint32_t l1 = 0, top = 0;                      // (l1: of a row that is not bad at most 32 x 2^23)
        out = 0;
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
                    out += a >= (uint32_t)Q_ROT_LIMIT ? 1 : 0;
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
        double b1 = (double)l1 * kc_absmax;
        b1 += __shfl_xor(b1, 16);
        b1 += __shfl_xor(b1, 32);
        bad = row_or<16>(top > 0x7F7F7Fu ? 1u : 0u) != 0 || !(b1 < DOT_MAX);
        check = !bad && !(b1 * 32768.0 < NARROW_LIMIT);
    }
};

// A step's keys: J tiles of 16 tokens, lane = (token, D / 4 channels), and the norms of the lane's own 4 tokens.
template <int D, int KB, int R>
struct Keys {
    static constexpr int J = 16 / R;
    Codes<D, KB> c[J];
    uint4 norms;                                       // (k, v) int16 each
    // Tiles past the span's last are that one again (and are not looked at). Rows up to a tile's end are
    // read whatever the sequence's length: a plane holds a multiple of 256.
    __device__ __forceinline__ void load(const Place<R> &p, const uint8_t *hb, const uint8_t *nb, int64_t span, int64_t u, int64_t last) {
        const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int64_t v = u + 16 * j < last ? u + 16 * j : last;
            c[j].load(hb, span, p.at(v) + col, grp);
        }
        const int64_t v = u + 16 * (col / R) < last ? u + 16 * (col / R) : last;
        norms = *(const uint4 *)(nb + (p.at(v) + 4 * grp) * 4);
    }
};

template <int D, int NC, int R, int FW>
struct Lds {
    static constexpr int J = 16 / R, RS = D == 64 ? 60 : 116;       // (the widest row: 4-bit keys, 3-bit values)
    static constexpr int SCORED = FW > 8 ? 7 : D == 128 && R == 16 ? 8 : 10;      // steps of a wave whose scores are kept
    static constexpr int FIRST = FW * R;               // runs: the first of each (span, row), and others
    static constexpr int NEAR = FIRST + (D == 64 ? (R == 16 ? 32 : 96) : (R == 16 ? 8 : R == 8 ? 24 : 48));
    alignas(16) v4i q[J][3][D / 64][64];
    union {
        alignas(16) int4 score[FW][SCORED][64];
        SerialLds<RS> fb[FW];
    } u;
    alignas(16) uint4 meta[NEAR];
    alignas(16) int32_t S[NEAR][D];
    alignas(16) uint32_t dig[3][4];
    uint16_t lut[LUT_N + 7];
    int32_t top[FW][R];
    uint32_t ev[FW][R];
    float bound[FW][R];                                // of the sum of |terms| of a span
    uint32_t qbad, over, check, pool, fail;            // rows as bits; runs taken
    unsigned long long events, bad, ovf, acc, score_max, range;
};

// FW: waves a workgroup.
template <int D, int KB, int NC, int R, int FW>
__global__ void __launch_bounds__(FW * 64, FW / 4) span_kernel(Job J) {
    using L = Lds<D, NC, R, FW>;
    constexpr int JT = L::J, ST = 16 * JT, CT = D / 16, PVK = NC / 4;
    __shared__ L S;
    Place<R> p(J);
    const Geom &g = J.g;
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, grp = lane >> 4, mine = col / R, r = col % R;
    // the lane's row, and what the tables are made of: requested together
    const int row = p.row0 + r < J.rows ? p.row0 + r : J.rows - 1;
    Query<D, KB> Q;
    if (wv < JT) Q.fetch(J.w.q + p.query(J, row) * D + grp * (D / 4));
    const int32_t kc = (int32_t)J.tabs->kc[tid & 15], ex = J.tabs->exp_table[tid & 255];
    p.find(J);
    const uint8_t *hb = plane_ptr(g, p.seq, p.kvh, 0), *nb = hb + (g.n_planes - 1) * g.span;
    // the wave's span, in tiles of 16
    const int nt = (int)((p.U + 15) >> 4), cut = span_start<FW>(nt, J.w.two_pass ? 0.0f : EVENTS);
    const int64_t lo = 16 * (int64_t)__builtin_amdgcn_readlane(cut, wv), stop = 16 * (int64_t)__builtin_amdgcn_readlane(cut, wv + 1);
    const int64_t hi = stop < p.U ? stop : p.U, last = (hi - 1) & ~(int64_t)15;
    Keys<D, KB, R> next;
    if (lo < hi) next.load(p, hb, nb, g.span, lo, last);
    const int64_t end = p.end(J, row), wlo = end - J.w.window;
    if (wv < JT) Q.make(J.kc_absmax);

    // -- tables ------------------------------------------------------------------------------
    if (tid == 0) {
        S.over = S.pool = S.fail = 0;
        S.events = S.bad = S.ovf = S.acc = S.score_max = 0;
    }
    if (tid < 256) {
#pragma unroll
        for (int i = 0; i < LUT_SPAN / 256; ++i) S.lut[256 * i + tid] = (uint16_t)(ex >> i);
        if (tid == 0) S.lut[LUT_SPAN] = 0;
    }
    if (tid < 16) {                                    // (no code names a centroid behind the codebook's end)
        const uint32_t z = balanced(kc);
#pragma unroll
        for (int l = 0; l < 3; ++l) ((uint8_t *)S.dig[l])[tid] = (uint8_t)(z >> (8 * l));
    }
    if (wv < JT) {
#pragma unroll
        for (int l = 0; l < 3; ++l)
#pragma unroll
            for (int b = 0; b < D / 64; ++b) S.q[wv][l][b][lane] = mine == wv ? Q.qd[l][b] : v4i{0, 0, 0, 0};
    }
    if (wv == 0) {
        const bool there = p.row0 + r < J.rows;
        const uint32_t bad = (uint32_t)__ballot(there && Q.bad), check = __ballot(there && Q.check) != 0;
        const int64_t out = J.count ? wave_sum_i64(there && mine == 0 ? Q.out : 0) : 0;
        if (lane == 0) {
            S.qbad = bad & ((1u << R) - 1u);
            S.check = check;
            S.range = (unsigned long long)out;
        }
    }
    __syncthreads();
    uint32_t dg[3][4];
#pragma unroll
    for (int i = 0; i < 3; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) dg[i][j] = (uint32_t)uni32((int)S.dig[i][j]);

    const bool check = uni32((int)S.check) != 0;
    const uint32_t qbad = (uint32_t)uni32((int)S.qbad);      // (such a row is taken to see nothing)
    // which of the lane's 4 tokens of the step its row sees, a bit each
    auto visible = [&](int64_t u) __attribute__((always_inline)) -> uint32_t {
        const int64_t t = p.at(u + 16 * mine) + 4 * grp;
        auto bits = [&](int64_t e) {                   // those below e
            const int64_t k = e - t;
            return k <= 0 ? 0u : k >= 4 ? 15u : (1u << (int)k) - 1u;
        };
        return (qbad >> r & 1u) != 0 || u + 16 * mine >= hi ? 0u : (~bits(wlo) | bits(J.w.sinks)) & bits(end);
    };
    // whether a row may not see all of a step
    auto edge = [&](int64_t u) __attribute__((always_inline)) {
        const int64_t t = p.at(u), e = p.at(u + ST - 16) + 16;
        return qbad != 0 || u + ST > hi || e > p.first_end || (t < p.last_lo && e > J.w.sinks);
    };
    // floor(dot k_norm / 2^24) of the lane's row and 4 tokens: dot = 2^16 H + L. Returns whether a visible one left int32
    auto scores = [&](const Keys<D, KB, R> &k, int64_t u, bool check, uint32_t in, int32_t (&s)[4]) __attribute__((always_inline)) {
        v4i T[5];
#pragma unroll
        for (int i = 0; i < 5; ++i) T[i] = v4i{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < JT; ++j) {
            if (j > 0 && u + 16 * j >= hi) break;
#pragma unroll
            for (int b = 0; b < D / 64; ++b) {
                v4i a[3], q[3];
#pragma unroll
                for (int l = 0; l < 3; ++l) q[l] = S.q[j][l][b][lane];
                expand16<KB>(k.c[j].bits(b, grp), dg, a);
#pragma unroll
                for (int l = 0; l < 3; ++l)
#pragma unroll
                    for (int i = 0; i < 3; ++i) T[l + i] = mma(a[l], q[i], T[l + i]);
            }
        }
        const uint32_t nw[4] = {k.norms.x, k.norms.y, k.norms.z, k.norms.w};
        bool over = false;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int32_t kn = (int16_t)(uint16_t)nw[i];
            const int32_t H = (int32_t)(((((uint32_t)T[4][i] << 8) + (uint32_t)T[3][i]) << 8) + (uint32_t)T[2][i]);
            const int32_t Lo = (int32_t)(((uint32_t)T[1][i] << 8) + (uint32_t)T[0][i]);
            const int64_t x = (int64_t)H * kn + (((int64_t)Lo * kn) >> 16);    // floor(dot k_norm / 2^16)
            s[i] = (int32_t)(uint32_t)((uint64_t)x >> 8);
            if (check) over |= ((x >> 8) != (int64_t)s[i] || s[i] == NONE) && (in >> i & 1) != 0;
        }
        return over;
    };

    // -- the scores ----------------------------------------------------------------------------
    int32_t m = NONE;
    {
        int32_t lowest = 0;
        bool over = false;
        int step = 0;
        for (int64_t u = lo; u < hi; u += ST, ++step) {
            const Keys<D, KB, R> cur = next;
            if (u + ST < hi) next.load(p, hb, nb, g.span, u + ST, last);
            int32_t s[4];
            uint32_t in = 15u;
            const bool e = edge(u);
            if (e) in = visible(u);
            over |= scores(cur, u, check, in, s);
            if (e) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool on = in >> i & 1;
                    lowest = on ? imin(lowest, s[i]) : lowest;
                    s[i] = on ? s[i] : NONE;
                }
            } else {
                lowest = imin(lowest, imin(imin(s[0], s[1]), imin(s[2], s[3])));
            }
            m = imax(m, imax(imax(s[0], s[1]), imax(s[2], s[3])));
            if (step < L::SCORED) S.u.score[wv][step][lane] = make_int4(s[0], s[1], s[2], s[3]);
        }
        if (over) atomicOr(&S.over, 1u << r);
        m = row_max<R>(m);
        if (grp == 0 && mine == 0) S.top[wv][r] = m;
        if (J.count && lo < hi && !over && p.row0 + r < J.rows && !(qbad >> r & 1u)) {
            const int64_t a = m == NONE ? 0 : m < 0 ? -(int64_t)m : m, c = -(int64_t)lowest;
            atomicMax(&S.score_max, (unsigned long long)(a > c ? a : c));
        }
    }
    // the lane's value words: CT codes together, of the field's words w0 and, over its end, w0 + 1
    const int bit = col * CT * g.vb, w0 = bit >> 5, sh = bit & 31;
    const int w1 = imin(w0 + 1, g.value_bytes / 4 - 1);
    const int pv = (g.key_bytes + 15) / 16;
    const uint8_t *const va0 = hb + (pv + w0 / 4) * g.span + (w0 % 4) * 4, *const va1 = hb + (pv + w1 / 4) * g.span + (w1 % 4) * 4;
    const int vw0 = imin(16, g.value_bytes - w0 / 4 * 16), vw1 = imin(16, g.value_bytes - w1 / 4 * 16);
    uint32_t vw[JT][4][NC == 8 ? 2 : 1];
    uint4 vnorm;
    auto values = [&](int64_t u) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < JT; ++j) {
            const int64_t t = p.at(u + 16 * j < last ? u + 16 * j : last) + 4 * grp;
            const uint8_t *const x = va0 + t * vw0, *const y = va1 + t * vw1;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                vw[j][i][0] = *(const uint32_t *)(x + i * vw0);
                if constexpr (NC == 8) vw[j][i][NC / 8] = *(const uint32_t *)(y + i * vw1);
            }
        }
        const int64_t t = u + 16 * mine < last ? u + 16 * mine : last;
        vnorm = *(const uint4 *)(nb + (p.at(t) + 4 * grp) * 4);
    };
    if (lo < hi) values(lo);                           // (in flight past the barrier)
    lds_barrier();

    // -- the walk ------------------------------------------------------------------------------
    const int64_t wg = blockIdx.x;
    uint4 *const far_meta = J.meta + wg * J.extra;
    int32_t *const far_S = J.S + wg * J.extra * D;
    if (lo < hi) {
        m = NONE;
        for (int i = 0; i < (J.w.two_pass ? FW : wv); ++i) m = imax(m, S.top[i][r]);
        double vcs[NC];
#pragma unroll
        for (int i = 0; i < NC; ++i) vcs[i] = J.vcs[i];
        const double vcmax = J.vcmax;
        const uint32_t delta_max = J.delta_max, wide = J.wide;
        bool first = wv == 0;                          // what the span finds is nothing: it scales in place
        // the run's digit sums, lane = (row, 4 channels a product) in the columns of the first group of tokens (the others'
        // take another group's terms with these codes, and are not read)
        v4i T[CT][3];
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
            for (int l = 0; l < 3; ++l) T[c][l] = v4i{0, 0, 0, 0};
        uint32_t lp = 0;                               // the lane's part of the denominator since the last event
        uint32_t l0 = 0;                               // first span: the row's denominator up to there
        float bs = 0.0f;                               // the lane's part of sum |v_norm p|
        const float bs_max = 0x1p28f / JT / (float)fmax(vcmax, 0x1p-23);  // (4 J lanes: terms below 2^30, and a step's 2^29)
        uint32_t wmax = 0, n_ev = 0;
        bool bad = false;
        int slot = wv * R + r, run = 0;                // the row's open run (-1: none was left); its tokens
        uint32_t fopen = 1u << PROB_FRAC;

        auto lut = [&](uint32_t d) __attribute__((always_inline)) -> uint32_t {
            return S.lut[__umulhi(d, (uint32_t)LOG2E_Q16 << 8)];        // floor(d log2(e) / 2^24), d <= delta_max
        };
        auto clip = [&](int32_t a, int32_t b) __attribute__((always_inline)) -> uint32_t {
            const uint32_t w = (uint32_t)a - (uint32_t)b;
            return w < delta_max ? w : delta_max;
        };
        // the run's sums: T[c][0] takes them
        auto gather = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    T[c][0][i] = (int)((((uint32_t)T[c][2][i] << 8) + (uint32_t)T[c][1][i]) * 256u + (uint32_t)T[c][0][i]);
                    T[c][1][i] = T[c][2][i] = 0;
                }
        };
        // (behind gather) the open run of the rows where `has`: into its record
        float bs_all = 0.0f;                           // a bound of the row's sums |terms| so far
        auto hand_over = [&](bool has, int to) __attribute__((always_inline)) {
            const uint32_t Ls = row_sum<R>(lp + (grp == 0 && mine == 0 ? l0 : 0u));
            float b = bs;
            if constexpr (R <= 4) b += __uint_as_float(xor_lane32<4>(__float_as_uint(b), lane));
            if constexpr (R <= 8) b += __uint_as_float(xor_lane32<8>(__float_as_uint(b), lane));
            b += __uint_as_float(xor_lane32<16>(__float_as_uint(b), lane));
            b += __uint_as_float(xor_lane32<32>(__float_as_uint(b), lane));
            b = b * (float)vcmax * 1.001f + (float)(RUN_MAX + ST);
            bs_all += has ? b : 0.0f;
            if (!has || slot < 0) return;
            const bool used = Ls != 0 || fopen != 1u << PROB_FRAC;
            const uint4 mt = make_uint4(Ls, fopen | (used ? USED : 0u), (uint32_t)to, __float_as_uint(b));
            const bool near = slot < L::NEAR;
            if (grp == 0 && mine == 0) {
                if (near)
                    S.meta[slot] = mt;
                else
                    far_meta[slot - L::NEAR] = mt;
            }
            if (!used || mine != 0) return;
            int32_t *const dst = near ? &S.S[slot][0] : far_S + (int64_t)(slot - L::NEAR) * D;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int c = 0; c < CT; c += 4)
                    *(v4i *)(dst + (4 * grp + i) * CT + c) = v4i{T[c][0][i], T[c + 1][0][i], T[c + 2][0][i], T[c + 3][0][i]};
            }
        };
        int step = 0;
        for (int64_t u = lo; u < hi; u += ST, ++step) {
            int32_t s[4];
            if (step < L::SCORED) {
                const int4 x = S.u.score[wv][step][lane];
                s[0] = x.x, s[1] = x.y, s[2] = x.z, s[3] = x.w;
            } else {
                Keys<D, KB, R> k;
                k.load(p, hb, nb, g.span, u, last);
                scores(k, u, false, 0, s);
                if (edge(u)) {
                    const uint32_t in = visible(u);
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[i] = in >> i & 1 ? s[i] : NONE;
                }
            }
            const int32_t vn[4] = {(int32_t)vnorm.x >> 16, (int32_t)vnorm.y >> 16, (int32_t)vnorm.z >> 16, (int32_t)vnorm.w >> 16};
            const int32_t mx = imax(imax(s[0], s[1]), imax(s[2], s[3]));
            const uint64_t evl = __ballot(mx > m);
            const bool ends = u + ST >= hi;
            // (else every p is 0; the last step's run ends there all the same)
            if (ends || evl != 0 || __ballot((uint32_t)m - (uint32_t)mx < delta_max) != 0) {
            run += ST;
            const float bs0 = bs;
            uint32_t pw[4];
            v4i A[3][PVK];                             // the columns' digits
            auto weights = [&](const uint32_t (&dl)[4]) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < 4; ++i) pw[i] = s[i] == NONE ? 0u : lut(dl[i]);
            };
            // the terms for the weights; returns the largest |v_norm p|
            auto terms = [&](const uint32_t (&pp)[4]) __attribute__((always_inline)) -> uint32_t {
                uint32_t top = 0;
                double wd[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int32_t w = __mul24(vn[i], (int)pp[i]);
                    const uint32_t aw = magnitude(w);
                    top = aw > top ? aw : top;
                    bs += (float)aw;
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
            // T += the terms in A, those of a group of tokens turned into the first group's columns
            auto accumulate = [&](bool three, uint32_t mask) __attribute__((always_inline)) {
#pragma unroll
                for (int j = 0; j < JT; ++j) {
                    if (JT > 1 && __ballot(mine == j && mask != 0) == 0) continue;
                    v4i B[3][PVK];
                    const uint32_t on = group_of<R>(j, mask);
#pragma unroll
                    for (int l = 0; l < 3; ++l)
#pragma unroll
                        for (int k = 0; k < PVK; ++k)
#pragma unroll
                            for (int i = 0; i < 4; ++i) B[l][k][i] = (int)(group_of<R>(j, (uint32_t)A[l][k][i]) & on);
                    // the lane's codes of 4 tokens, in bytes or halves (the shift is opaque, so that the one-hot codes are
                    // made where they are used: kept over the segments' loop they take all registers there are)
                    int sh_ = sh;
                    asm volatile("" : "+v"(sh_));
                    uint32_t x[NC == 8 ? CT / 2 : CT / 4];
                    if constexpr (NC == 4) {
                        const uint32_t by = (uint32_t)sh_ >> 3, sel = by | (4u + by) << 8;
#pragma unroll
                        for (int h = 0; h < CT / 4; ++h) {
                            const uint32_t q = sel + 0x0101u * (uint32_t)(g.vb == 2 ? h : 0);
                            x[h] = perm(vw[j][1][0], vw[j][0][0], q | 0x0C0C0000u) | perm(vw[j][3][0], vw[j][2][0], q << 16 | 0x0C0Cu);
                        }
                        if (g.vb == 1) {
                            x[0] >>= sh_ & 7;
                            if constexpr (CT == 8) x[CT / 8] = x[0] >> 4;
                        }
                    } else {
#pragma unroll
                        for (int h = 0; h < CT / 4; ++h) {
                            uint32_t f[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const uint32_t hi_ = vw[j][i][NC / 8], lo_ = vw[j][i][0];
                                f[i] = __builtin_amdgcn_alignbit(hi_, lo_, sh_) >> (12 * h);
                            }
                            x[2 * h] = perm(f[1], f[0], 0x05040100u);
                            x[2 * h + 1] = perm(f[3], f[2], 0x05040100u);
                        }
                    }
#pragma unroll
                    for (int c = 0; c < CT; ++c) {
                        uint32_t codes;
                        if constexpr (NC == 4) {
                            codes = g.vb == 2 ? x[c / 4] >> (2 * (c % 4)) & 0x03030303u : x[c / 4] >> (c % 4) & 0x01010101u;
                        } else {
                            const uint32_t a = x[c / 4 * 2] >> (3 * (c % 4)) & 0x00070007u, b = x[c / 4 * 2 + 1] >> (3 * (c % 4)) & 0x00070007u;
                            codes = perm(b, a, 0x06040200u);
                        }
                        v4i oh[PVK];
#pragma unroll
                        for (int k = 0; k < NC; ++k)   // 1 where a code (bytes of 4) is k
                            oh[k / 4][k % 4] = (int)(k < 4 ? perm(0u, 1u << (8 * k), codes) : perm(1u << (8 * (k - 4)), 0u, codes));
#pragma unroll
                        for (int k = 0; k < PVK; ++k) {
                            T[c][0] = mma(oh[k], B[0][k], T[c][0]);
                            T[c][1] = mma(oh[k], B[1][k], T[c][1]);
                            if (three) T[c][2] = mma(oh[k], B[2][k], T[c][2]);
                        }
                    }
                }
            };
            // events: the row's tokens, in the order (group of tokens, lane group, token), fall into segments, one more
            // than its events (bits 8 i of seg the segment of token i)
            const uint32_t there = u + 16 * mine < hi ? ~0u : 0u;      // (the lane's tokens are the span's)
            uint32_t dl[4], fe[4] = {0, 0, 0, 0}, seg = 0;
            int row_ev = 0;
            if (evl == 0) {
#pragma unroll
                for (int i = 0; i < 4; ++i) dl[i] = clip(m, s[i]);
            } else {
                const int ord = 4 * mine + grp;
                auto from = [&](int32_t v, int o, int32_t none) __attribute__((always_inline)) {  // of the lane o before in that order
                    const int q = ord - o;
                    const int32_t x = __shfl(v, (q & 3) * 16 + (q >> 2) * R + r);
                    return q < 0 ? none : x;
                };
                int32_t e = mx;
#pragma unroll
                for (int o = 1; o < 4 * JT; o *= 2) e = imax(e, from(e, o, NONE));
                e = imax(m, from(e, 1, NONE));         // the maximum before the lane's tokens
                uint32_t n = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool ev = s[i] > e;
                    const uint32_t dd = clip(ev ? s[i] : e, ev ? e : s[i]);
                    fe[i] = ev ? dd + 1u : 0u;         // an event's distance, + 1
                    dl[i] = ev ? 0u : dd;
                    e = ev ? s[i] : e;
                    n += ev ? 1 : 0;
                    seg |= n << (8 * i);
                }
                uint32_t off = n;
#pragma unroll
                for (int o = 1; o < 4 * JT; o *= 2) off += (uint32_t)from((int32_t)off, o, 0);
                const int lastlane = 48 + (JT - 1) * R + r;
                row_ev = __shfl((int)off, lastlane);
                m = __shfl(e, lastlane);
                seg += (off - n) * 0x01010101u;        // at most 64
                n_ev += n;
            }
            weights(dl);
            const uint32_t top = terms(pw);
            wmax = top > wmax ? top : wmax;
            const bool three = __ballot(top > wide) != 0;
            const float bs_step = bs - bs0;            // (every run of the step is bounded by all of it)
            for (int sg = 0;; ++sg) {
                uint32_t mask = there;
                if (evl == 0) {
                    lp += (pw[0] + pw[1]) + (pw[2] + pw[3]);
                } else {                               // the segment's tokens, a byte each
                    mask = 0;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const bool now = ((seg >> (8 * i)) & 0xFFu) == (uint32_t)sg;
                        mask |= now ? 0xFFu << (8 * i) : 0u;
                        lp += now ? pw[i] : 0u;
                    }
                    mask &= there;
                }
                accumulate(three, mask);
                // the rows whose run ends: with an event, or all with the span, or before L or acc could leave 32 bits
                bool has = row_ev > sg;
                const bool event = __ballot(has) != 0;
                if (!event) {
                    if (!ends && run < RUN_MAX && __ballot(bs > bs_max) == 0) break;
                    has = true;
                }
                // the event opens segment sg + 1 of the row
                uint32_t fd = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) fd = ((seg >> (8 * i)) & 0xFFu) == (uint32_t)(sg + 1) && fe[i] ? fe[i] : fd;
                fd = row_or<R>(fd);
                const uint32_t f = has && event ? lut(fd - 1u) : 1u << PROB_FRAC;
                gather();
                if (event && first) {
                    const uint32_t l = l0 + row_sum<R>(lp);
                    if (has) {
#pragma unroll
                        for (int c = 0; c < CT; ++c) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                // floor(a f / 2^15) in halves of 16 bits: 2 hi f + floor(lo f / 2^15)
                                const int32_t a = T[c][0][i];
                                const uint32_t l16 = __umul24((uint32_t)a & 0xFFFFu, f) >> PROB_FRAC;
                                T[c][0][i] = __mul24(a >> 16, 2 * (int)f) + (int)l16;
                            }
                        }
                        l0 = (uint32_t)(((uint64_t)l * f) >> PROB_FRAC);
                        lp = 0;
                    }
                    continue;
                }
                // a row for which no run is left goes token by token and writes no more
                first = false;
                int to = -1;
                if (event || !ends) {
                    if (has && grp == 0 && mine == 0) to = (int)atomicAdd(&S.pool, 1u);
                    to = __shfl(to, r);
                    const bool none = L::FIRST + to >= L::NEAR + J.extra;
                    bad = bad || (has && none);
                    to = none ? -1 : L::FIRST + to;
                }
                hand_over(has, to);
                if (has) {
                    slot = to;
                    fopen = f;
                    lp = 0;
                    l0 = 0;
                    bs = event ? bs_step : 0.0f;
#pragma unroll
                    for (int c = 0; c < CT; ++c) T[c][0] = v4i{0, 0, 0, 0};
                }
                if (!event) {
                    run = 0;
                    break;
                }
            }
            }
            if (u + ST < hi) values(u + ST);           // the next step's values are requested
        }
        bad = bad || !((double)wmax * vcmax + 2.0 <= TERM_LIMIT);
        const uint32_t events = row_sum<R>(n_ev), any = row_or<R>(bad ? BAD : 0u);
        if (grp == 0 && mine == 0) {
            S.ev[wv][r] = events | any;
            S.bound[wv][r] = bs_all;
        }
    } else if (grp == 0 && mine == 0) {                // (a span without tokens)
        S.meta[wv * R + r] = make_uint4(0, 1u << PROB_FRAC, ~0u, 0);
        S.ev[wv][r] = 0;
        S.bound[wv][r] = 0.0f;
    }
    __syncthreads();

    // -- the runs: a wave a row, lane = channel ----------------------------------------------------
    const int ns = imin(nt, FW);
    for (int rr = wv; rr < R && p.row0 + rr < J.rows; rr += FW) {
        constexpr int CPL = D / 64;
        const uint32_t e = lane < ns ? S.ev[lane][rr] : 0u;
        const uint4 mine_ = S.meta[(lane < ns ? lane : 0) * R + rr];   // lane i: the first run of span i
        bool wrong = __ballot((e & BAD) != 0) != 0 || ((qbad | S.over) >> rr & 1u) != 0;
        int64_t acc[CPL];                              // (online: what 32 bits hold)
        uint64_t l = 0;
#pragma unroll
        for (int k = 0; k < CPL; ++k) acc[k] = 0;
        // of a run that is not in LDS' first ones, or follows one of them
        uint4 mt;
        int32_t v[CPL];
        auto follow = [&](int slot) __attribute__((always_inline)) {
            if (slot < L::NEAR) {
                mt = S.meta[slot];
#pragma unroll
                for (int k = 0; k < CPL; ++k) v[k] = S.S[slot][lane + 64 * k];
            } else {
                mt = far_meta[slot - L::NEAR];
#pragma unroll
                for (int k = 0; k < CPL; ++k) v[k] = far_S[(int64_t)(slot - L::NEAR) * D + lane + 64 * k];
            }
        };
        auto scaled = [&](int32_t x, int32_t f) __attribute__((always_inline)) {       // floor(x f / 2^15)
            return __mul24(x >> 16, 2 * f) + (int32_t)(__umul24((uint32_t)x & 0xFFFFu, (uint32_t)f) >> PROB_FRAC);
        };
        float all = lane < ns ? S.bound[lane][rr] : 0.0f;
#pragma unroll
        for (int o = 1; o < 16; o *= 2) all += __shfl_xor(all, o);
        if (wrong) {
        } else if (uni32(all <= 2147483000.0f)) {
            // no |acc| on the way passes the sum of all |terms|: 32 bits, no clamp
            int32_t a32[CPL], v2[CPL];
#pragma unroll
            for (int k = 0; k < CPL; ++k) {
                a32[k] = 0;
                v2[k] = S.S[rr][lane + 64 * k];
            }
            // (the loops are not unrolled: their instructions come from memory but once)
#pragma unroll 1
            for (int i = 0; i < ns; ++i) {
                const int after = i + 1 < ns ? i + 1 : i;
#pragma unroll
                for (int k = 0; k < CPL; ++k) {
                    v[k] = v2[k];
                    v2[k] = S.S[after * R + rr][lane + 64 * k];
                }
                uint32_t Lr = (uint32_t)__builtin_amdgcn_readlane((int)mine_.x, i), fr = (uint32_t)__builtin_amdgcn_readlane((int)mine_.y, i);
                int slot = __builtin_amdgcn_readlane((int)mine_.z, i);
#pragma unroll 1
                for (;;) {
                    if (fr & USED) {
                        const int32_t ff = (int32_t)(fr & (USED - 1));
                        if (ff != 1 << PROB_FRAC) {
#pragma unroll
                            for (int k = 0; k < CPL; ++k) a32[k] = scaled(a32[k], ff);
                            l = (l * (uint32_t)ff) >> PROB_FRAC;
                        }
#pragma unroll
                        for (int k = 0; k < CPL; ++k) a32[k] += v[k];
                        l += Lr;
                    }
                    if (slot < 0) break;
                    follow(slot);
                    Lr = (uint32_t)uni32((int)mt.x);
                    fr = (uint32_t)uni32((int)mt.y);
                    slot = uni32((int)mt.z);
                }
            }
#pragma unroll
            for (int k = 0; k < CPL; ++k) acc[k] = a32[k];
        } else {
#pragma unroll 1
            for (int i = 0; i < ns; ++i) {
#pragma unroll 1
                for (int slot = i * R + rr; slot >= 0;) {
                    follow(slot);
                    const uint32_t Lr = (uint32_t)uni32((int)mt.x), fr = (uint32_t)uni32((int)mt.y);
                    const float bound = __uint_as_float((uint32_t)uni32((int)mt.w));
                    slot = uni32((int)mt.z);
                    if (!(fr & USED)) continue;
                    const int32_t ff = (int32_t)(fr & (USED - 1));
#pragma unroll
                    for (int k = 0; k < CPL; ++k) {
                        if (!J.w.two_pass) {           // (two-pass: no factors; clamped once, at the end)
                            const int32_t y = scaled((int32_t)acc[k], ff);
                            wrong = wrong || !(fabsf((float)y) + bound <= 2147483000.0f);
                            acc[k] = y;
                        }
                        acc[k] += v[k];
                    }
                    l = (J.w.two_pass ? l : (l * (uint32_t)ff) >> PROB_FRAC) + Lr;
                }
            }
            wrong = __ballot(wrong) != 0;
        }
        if (wrong) {
            if (lane == 0) atomicOr(&S.fail, 1u << rr);
            continue;
        }
        const Recip rc = reciprocal((int64_t)l);
        const int64_t at = p.query(J, p.row0 + rr) * D;
        int64_t amax = 0, over = 0;
#pragma unroll
        for (int k = 0; k < CPL; ++k) {
            if (acc[k] < ACC_LO || acc[k] > ACC_HI) {
                ++over;
                acc[k] = acc[k] < ACC_LO ? ACC_LO : ACC_HI;
            }
            J.w.out[at + lane + 64 * k] = (int32_t)(wmul(acc[k], rc.r) >> rc.shift);
            const int64_t a = acc[k] < 0 ? -acc[k] : acc[k];
            amax = a > amax ? a : amax;
        }
        if (J.count) {
            const int64_t ev = wave_sum_i64((int64_t)(e & ~BAD));
            amax = wave_max_i64(amax);
            over = wave_sum_i64(over);
            if (lane == 0) {
                if (ev && !J.w.two_pass) atomicAdd(&S.events, (unsigned long long)ev);
                if (over) atomicAdd(&S.ovf, (unsigned long long)over);
                atomicMax(&S.acc, (unsigned long long)amax);
            }
        }
    }
    __syncthreads();                                   // (the serial path's rows lie over the scores)
    const uint32_t fail = (uint32_t)uni32((int)S.fail);
    for (int rr = wv; rr < R; rr += FW) {
        if (!(fail >> rr & 1u)) continue;
        const int64_t at = p.query(J, p.row0 + rr) * D, T_ = p.end(J, p.row0 + rr);
        serial_head<D / 64, L::RS>(g, J.tabs, J.tabs->kc, J.tabs->vc, J.w.q + at, p.seq, p.kvh, T_, J.w.two_pass, true, S.u.fb[wv],
                                   J.w.out + at, J.st, rows_of(J.w, T_));
        if (lane == 0) atomicAdd(&S.bad, 1ull);
    }
    if (!J.count) return;
    __syncthreads();
    if (tid == 0) {
        DevStats *const st = J.st;
        if (S.events) atomicAdd(&st->rescale_events, S.events);
        if (S.bad) atomicAdd(&st->serial_fallbacks, S.bad);
        if (S.ovf) atomicAdd(&st->acc_overflows, S.ovf);
        if (S.range) atomicAdd(&st->range_errors, S.range);
        if (S.acc > st->max_abs_acc) atomicMax(&st->max_abs_acc, S.acc);
        if (S.score_max > st->max_abs_score) atomicMax(&st->max_abs_score, S.score_max);
        if (p.kvh == 0 && p.row0 + R >= J.rows) {
            const int64_t T_ = p.base + J.w.n;
            atomicMax(&st->n_tokens, (unsigned long long)rows_of(J.w, T_).count(T_));
        }
    }
}

// Any format, token by token: a wave a (query, head).
constexpr int SERIAL_RS = 272;   // >= the widest row (8b/8b at d = 128: 260 B)
template <int CPL>
__global__ void __launch_bounds__(64) serial_kernel(Geom g, const Tables *__restrict__ tabs, WindowJob w, DevStats *st) {
    __shared__ int64_t kc[256], vc[256];
    __shared__ __align__(16) SerialLds<SERIAL_RS> L;
    const int lane = threadIdx.x;
    const int qh = (int)(blockIdx.x % (unsigned)g.n_q);
    const int64_t rest = blockIdx.x / (unsigned)g.n_q;
    const int64_t i = rest % w.n;
    const int b = w.seq_lo + (int)(rest / w.n);
    for (int j = lane; j < (1 << g.kb); j += 64) kc[j] = tabs->kc[j];
    for (int j = lane; j < (1 << g.vb); j += 64) vc[j] = tabs->vc[j];
    const int64_t at = (int64_t)blockIdx.x * g.d;
    for (int c = lane; c < g.d; c += 64) {
        const int64_t x = w.q[at + c];
        if (x >= Q_ROT_LIMIT || x <= -Q_ROT_LIMIT) atomicAdd(&st->range_errors, 1ull);
    }
    __syncthreads();
    const int64_t T = end_of(w, b, i);
    serial_head<CPL, SERIAL_RS>(g, tabs, kc, vc, w.q + at, b, qh / g.G, T, w.two_pass, true, L, w.out + at, st, rows_of(w, T));
}

namespace {
// rows a tile: as many as there are, up to 16
int tile_rows(int64_t rows) { return rows <= 4 ? 4 : rows <= 8 ? 8 : 16; }
int64_t workgroups(const Geom &g, int64_t n, int64_t nseq) {
    const int64_t rows = n * g.G, R = tile_rows(rows);
    return nseq * g.n_kv * ((rows + R - 1) / R);
}
constexpr int64_t LAUNCH = 1024;                       // workgroups a launch, which bounds the scratch
// runs a workgroup has in the scratch beside those in LDS: up to 1,024 in 16 MiB, but 192 at least. (Random scores take a
// tile of 16 rows some 60 over 4,096 rows; one that is out of runs goes token by token, at 100 times the cost.)
int64_t extra_runs(const Geom &g, int64_t wgs) {
    return std::max<int64_t>(192, std::min<int64_t>(1024, ((int64_t)16 << 20) / (wgs * (g.d * 4 + 16))));
}
}  // namespace

template <int D, int KB, int NC>
hipError_t launch(hipStream_t s, const Job &J, unsigned blocks, LaunchEv ev) {
    const int R = tile_rows(J.rows);
    constexpr int FW = D == 64 && NC == 4 ? 12 : 8;
    if (R == 4)
        hipExtLaunchKernelGGL((span_kernel<D, KB, NC, 4, FW>), dim3(blocks), dim3(FW * 64), 0, s, ev.start, ev.stop, 0, J);
    else if (R == 8)
        hipExtLaunchKernelGGL((span_kernel<D, KB, NC, 8, FW>), dim3(blocks), dim3(FW * 64), 0, s, ev.start, ev.stop, 0, J);
    else
        hipExtLaunchKernelGGL((span_kernel<D, KB, NC, 16, FW>), dim3(blocks), dim3(FW * 64), 0, s, ev.start, ev.stop, 0, J);
    return hipGetLastError();
}

}  // namespace wn

int64_t window_tiles(const Geom &g, int64_t n, int64_t nseq) { return wn::workgroups(g, n, nseq); }

size_t window_scratch_bytes(const Geom &g, int64_t n, int64_t nseq) {
    const int64_t wgs = std::min(wn::workgroups(g, n, nseq), wn::LAUNCH), runs = wgs * wn::extra_runs(g, wgs);
    return (size_t)runs * (16 + g.d * 4) + 256;
}

hipError_t launch_attend_window_spans(hipStream_t s, const Geom &g, const Tables *t, const Tables &host, const WindowJob &w, bool count,
                                      void *scratch, size_t scratch_bytes, LaunchEv ev, DevStats *st) {
    using namespace wn;
    Job J{};
    const int64_t all = workgroups(g, w.n, w.nseq), wgs = std::min(all, LAUNCH);
    if (all > 0x7fffffff || window_scratch_bytes(g, w.n, w.nseq) > scratch_bytes) return hipErrorInvalidValue;
    J.g = g;
    J.tabs = t;
    J.w = w;
    J.rows = (int32_t)(w.n * g.G);
    J.chains = w.nseq * g.n_kv;
    J.extra = (int32_t)extra_runs(g, wgs);
    J.count = count ? 1 : 0;
    J.kc_absmax = host.kc_absmax;
    for (int i = 0; i < 1 << g.vb; ++i) {
        J.vcs[i] = (double)host.vc[i] * 0x1p-23;
        J.vcmax = std::fmax(J.vcmax, std::fabs(J.vcs[i]));
    }
    J.wide = (uint32_t)(32639.0 / std::fmax(J.vcmax, 0x1p-16));
    J.delta_max = (uint32_t)host.delta_max;
    J.meta = (uint4 *)scratch;
    J.S = (int32_t *)((uint8_t *)scratch + (wgs * J.extra * 16 + 255) / 256 * 256);
    J.st = st;
    hipError_t (*run)(hipStream_t, const Job &, unsigned, LaunchEv) = nullptr;
#define INSITU_WINDOW_CASE(DD, KK, CC) \
    if (g.d == DD && g.kb == KK && (g.vb <= 2 ? 4 : 8) == CC) run = launch<DD, KK, CC>;
#define INSITU_WINDOW_D(DD)                                                                           \
    INSITU_WINDOW_CASE(DD, 2, 4) INSITU_WINDOW_CASE(DD, 3, 4) INSITU_WINDOW_CASE(DD, 4, 4)            \
    INSITU_WINDOW_CASE(DD, 2, 8) INSITU_WINDOW_CASE(DD, 3, 8) INSITU_WINDOW_CASE(DD, 4, 8)
    INSITU_WINDOW_D(64)
    INSITU_WINDOW_D(128)
#undef INSITU_WINDOW_D
#undef INSITU_WINDOW_CASE
    if (!run) return hipErrorInvalidValue;
    for (int64_t first = 0; first < all; first += LAUNCH) {
        J.first = (uint32_t)first;
        const LaunchEv e{first == 0 ? ev.start : nullptr, first + LAUNCH >= all ? ev.stop : nullptr};
        const hipError_t rc = run(s, J, (unsigned)std::min(all - first, LAUNCH), e);
        if (rc != hipSuccess) return rc;
    }
    return hipSuccess;
}

hipError_t launch_attend_window_serial(hipStream_t s, const Geom &g, const Tables *t, const WindowJob &w, LaunchEv ev,
                                       DevStats *st) {
    const int64_t blocks = w.nseq * w.n * g.n_q;
    if (blocks > 0x7fffffff) return hipErrorInvalidValue;
    if (g.d <= 64)
        hipExtLaunchKernelGGL(wn::serial_kernel<1>, dim3((unsigned)blocks), dim3(64), 0, s, ev.start, ev.stop, 0, g, t, w, st);
    else
        hipExtLaunchKernelGGL(wn::serial_kernel<2>, dim3((unsigned)blocks), dim3(64), 0, s, ev.start, ev.stop, 0, g, t, w, st);
    return hipGetLastError();
}

}  // namespace insitu
