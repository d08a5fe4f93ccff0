// Rows of a cache moved between and within its sequences: forks (one sequence's rows, whole or with
// a selection of the last ones, to others) and the compaction of a sequence's last rows (the accepted
// path of a draft). The reference's cache holds one sequence and only appends (cache/base.py:29-81);
// the rows' bytes and planes are its own (hw/ddr_layout.py:148-214).
//
// Both are copies, bound by memory: every byte of a row is read once, and once for all copies of it. A
// lane takes 16 bytes of a destination plane, which in the narrower planes (8 and 4 bytes a row) are
// the pieces of 2 or 4 rows, one load where those lie together in the source and one a row where not.
// Measured: 8 copies of 32,768 rows (8 heads, 4b/2b, 123 MB with what is read) 25 us, 4.9 TB/s, as a large
// copy; 14,003 of the last 30,001 rows at d = 128 12 us for 27 MB (every other row kept: the lines of the
// others are read with it); 3 copies of 100 rows 5 us, a launch.
#include "insitu_internal.h"

namespace insitu {
namespace {

__device__ __forceinline__ int64_t source_row(const RowCopy &c, int64_t r, int z) {
    if (r < c.head[z]) return r;
    const int64_t j = r - c.head[z];
    if (!c.rows) return c.add[z] + j;
    // (a row outside the selection's range would leave the sequence: the nearest one inside)
    int64_t i = c.rows[(int64_t)c.rows_at[z] * c.rows_stride + j];
    i = i < 0 ? 0 : i;
    return c.add[z] + (i < c.n ? i : c.n - 1);
}

constexpr int UNITS = 4;       // 16-byte units a lane, their loads in flight together

__global__ void __launch_bounds__(256) copy_rows_kernel(Geom s, Geom t, RowCopy c) {
    const int z = blockIdx.z, p = blockIdx.y % s.n_planes, h = blockIdx.y / s.n_planes;
    if (blockIdx.x == 0 && blockIdx.y == 0 && c.len[0] && threadIdx.x < (unsigned)(c.first[z + 1] - c.first[z]))
        for (int64_t *len : c.len) len[c.dst[c.first[z] + threadIdx.x]] = c.end[z];
    const int w = s.plane_w[p], per = 16 / w;
    const int64_t begin = c.begin[z], end = c.end[z];
    const int64_t u0 = begin / per, u1 = (end + per - 1) / per;
    const int64_t first = u0 + (int64_t)blockIdx.x * (256 * UNITS) + threadIdx.x;
    if (u0 + (int64_t)blockIdx.x * (256 * UNITS) >= u1) return;
    const uint8_t *src = plane_ptr(s, c.src[z], h, p);
    uint4 v[UNITS];
#pragma unroll
    for (int i = 0; i < UNITS; ++i) {
        const int64_t u = first + 256 * i;
        v[i] = make_uint4(0u, 0u, 0u, 0u);
        if (u >= u1) continue;
        const int64_t r = u * per;
        if (w == 16) {
            v[i] = *(const uint4 *)(src + source_row(c, r, z) * 16);
        } else if (r + per <= c.head[z]) {
            v[i] = *(const uint4 *)(src + r * w);
        } else if (w == 8) {
            const uint2 a = r >= begin && r < end ? *(const uint2 *)(src + source_row(c, r, z) * 8) : make_uint2(0u, 0u);
            const uint2 b = r + 1 >= begin && r + 1 < end ? *(const uint2 *)(src + source_row(c, r + 1, z) * 8) : make_uint2(0u, 0u);
            v[i] = make_uint4(a.x, a.y, b.x, b.y);
        } else if (w == 4) {
            uint32_t x[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
                x[k] = r + k >= begin && r + k < end ? *(const uint32_t *)(src + source_row(c, r + k, z) * 4) : 0u;
            v[i] = make_uint4(x[0], x[1], x[2], x[3]);
        }
    }
    for (int k = c.first[z]; k < c.first[z + 1]; ++k) {
        uint8_t *dst = plane_ptr(t, c.dst[k], h, p);
#pragma unroll
        for (int i = 0; i < UNITS; ++i) {
            const int64_t u = first + 256 * i, r = u * per;
            if (u >= u1) continue;
            if (r >= begin && r + per <= end) {
                *(uint4 *)(dst + u * 16) = v[i];
                continue;
            }
            // the rows at either end, one by one: their neighbours are not this call's
            const uint32_t x[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                const int64_t rd = r + 4 * d / w;
                if (rd >= begin && rd < end) *(uint32_t *)(dst + u * 16 + 4 * d) = x[d];
            }
        }
    }
}

// Up to 1,024 kept rows of a sequence's last n: a workgroup a (plane, KV head, sequence) reads them
// all before it writes one, so that it may write where it reads (1,024 rows 4 to 7 us; more go through a
// buffer, two launches a sequence: 1,025 rows of one sequence 15 us, of 16 sequences 200).
__global__ void __launch_bounds__(1024) keep_rows_kernel(Geom g, RowKeep c) {
    const int p = blockIdx.x, h = blockIdx.y, z = blockIdx.z, b = c.seq0 + z;
    const int j = threadIdx.x, count = c.count[z];
    const int64_t base = c.base[z];
    if (p == 0 && h == 0 && j == 0)
        for (int64_t *len : c.len) len[b] = base + count;
    const int w = g.plane_w[p];
    uint8_t *rows = plane_ptr(g, b, h, p) + base * w;
    int i = j < count ? c.rows[(int64_t)b * c.rows_stride + j] : 0;
    i = i < 0 ? 0 : i < c.n ? i : c.n - 1;
    const uint32_t *src = (const uint32_t *)(rows + (int64_t)i * w);
    uint32_t x[4] = {0u, 0u, 0u, 0u};
    if (j < count) {
        if (w == 16) {
            const uint4 v = *(const uint4 *)src;
            x[0] = v.x;
            x[1] = v.y;
            x[2] = v.z;
            x[3] = v.w;
        } else {
            x[0] = src[0];
            if (w >= 8) x[1] = src[1];
        }
    }
    __syncthreads();
    if (j >= count || i == j) return;
    uint32_t *dst = (uint32_t *)(rows + (int64_t)j * w);
    if (w == 16) {
        *(uint4 *)dst = make_uint4(x[0], x[1], x[2], x[3]);
    } else {
        dst[0] = x[0];
        if (w >= 8) dst[1] = x[1];
    }
}

}  // namespace

hipError_t launch_copy_rows(hipStream_t s, const Geom &src, const Geom &dst, const RowCopy &c, int groups) {
    int64_t units = 0;
    for (int z = 0; z < groups; ++z) {
        const int64_t u = c.end[z] - c.begin[z] + 1;             // (a unit more where begin and end share none)
        units = u > units ? u : units;
    }
    const int64_t blocks = (units + 256 * UNITS - 1) / (256 * UNITS);
    hipLaunchKernelGGL(copy_rows_kernel, dim3((unsigned)(blocks > 0 ? blocks : 1), (unsigned)(src.n_planes * src.n_kv), (unsigned)groups),
                       dim3(256), 0, s, src, dst, c);
    return hipGetLastError();
}

hipError_t launch_keep_rows(hipStream_t s, const Geom &g, const RowKeep &c, int seqs, int most) {
    hipLaunchKernelGGL(keep_rows_kernel, dim3((unsigned)g.n_planes, (unsigned)g.n_kv, (unsigned)seqs),
                       dim3((unsigned)(most > 64 ? (most + 63) / 64 * 64 : 64)), 0, s, g, c);
    return hipGetLastError();
}

}  // namespace insitu
