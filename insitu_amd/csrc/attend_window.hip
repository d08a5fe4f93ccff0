// The attend of layers with a sliding window (and a few first rows that stay visible): the last n rows of a
// sequence are the queries' own, and the query at row p attends, in row order, the rows t <= p with t < sinks
// or t > p - window, with the integers that attend_online / attend_two_pass (ops/attention.py:429-513) give
// on those rows. The reference attends all of a context and has no counterpart.
#include "serial_head.h"

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

}  // namespace wn

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
