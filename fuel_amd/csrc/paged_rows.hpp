// Attention of few rows a sequence over a paged KV cache: the walk over the keys
// of a batch in tiles of 16 query rows, for caches of any element type.  A, the
// accumulator of a wavefront, brings the type's loads and products (paged.hip,
// paged8.hip):
//   Cache, Row, DIM, VW   the cache's view, the rows' type, head_dim, DIM / 16
//   STEP, BYTES           keys of a block, which a wavefront takes at a time; bytes
//                         of a key or value row
//   RESIDENT              workgroups a CU
//   load_q, start, walk, walk_odd, finish;  o, m, l, limit
// Lane 16 g + r holds of query row r the dims VW (4 g + k) + t as o[t][k], the
// running maximum m, the sum l, and limit, the row's position.
#pragma once

#include <hip/hip_runtime.h>

#include "common.hpp"
#include "kernels.hpp"
#include "paged.hpp"

namespace frq {

constexpr int PA_WAVES = 4;

// The largest of the four lanes 16 g + r of a row, in all four.
__device__ __forceinline__ float pg_row_max(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const float w = fmaxf(__builtin_bit_cast(float, (uint32_t)a[0]), __builtin_bit_cast(float, (uint32_t)a[1]));
    const uint32_t x = __builtin_bit_cast(uint32_t, w);
    const auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return fmaxf(__builtin_bit_cast(float, (uint32_t)b[0]), __builtin_bit_cast(float, (uint32_t)b[1]));
}

// A lane's query row as the operands of KS products: 8 elements of x from dim(t) on
// each, in NQ parts of type E, and the factor that makes scores in log2 units of
// their products.  16-bit rows are of type E.
template <class E, int NQ, int KS, class T, class Dim>
__device__ __forceinline__ void pd_load_q(typename PgElem<E>::v8 (&q)[NQ][KS], float& factor, const T* x, float scale,
                                          Dim dim) {
    using v8 = typename PgElem<E>::v8;
    // (negated for a negative scale: the maximum is taken of scores with a positive factor)
    factor = fabsf(scale) * 1.4426950408889634f;
    if constexpr (!std::is_same<T, float>::value) {
        const uint32_t flip = scale < 0.0f ? 0x80008000u : 0;
#pragma unroll
        for (int t = 0; t < KS; t++)
            q[0][t] = __builtin_bit_cast(v8, *reinterpret_cast<const pg_u4*>(x + dim(t)) ^ flip);
        return;
    }
    float f[KS][8];
#pragma unroll
    for (int t = 0; t < KS; t++) {
        T raw[8];
        __builtin_memcpy(raw, __builtin_assume_aligned(x + dim(t), 16), sizeof raw);
#pragma unroll
        for (int e = 0; e < 8; e++) f[t][e] = scale < 0.0f ? -(float)raw[e] : (float)raw[e];
    }
    if constexpr (std::is_same<E, _Float16>::value) {
        float a = 0.0f;
#pragma unroll
        for (int t = 0; t < KS; t++)
#pragma unroll
            for (int e = 0; e < 8; e++) a = fmaxf(a, fabsf(f[t][e]));
        a = fmaxf(a, __shfl_xor(a, 16));
        a = fmaxf(a, __shfl_xor(a, 32));
        // (a row with an infinite value keeps it; its scores are no numbers anyway)
        const int ex = a > 0.0f && a < __builtin_inff() ? max(-100, __builtin_amdgcn_frexp_expf(a) - 15) : 0;
#pragma unroll
        for (int t = 0; t < KS; t++)
#pragma unroll
            for (int e = 0; e < 8; e++) f[t][e] = __builtin_amdgcn_ldexpf(f[t][e], -ex);
        factor = __builtin_amdgcn_ldexpf(factor, ex);
    }
#pragma unroll
    for (int t = 0; t < KS; t++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
            float rest = f[t][e];
#pragma unroll
            for (int p = 0; p < NQ; p++) {
                q[p][t][e] = (E)rest;
                rest -= (float)q[p][t][e];
            }
        }
}

// ---- few rows a sequence ----
//
// The query rows of a sequence and KV head in tiles of 16, and for each tile
// the sequence's keys in units of `unit` keys, are one list (head by head,
// within a head sequence by sequence, tile by tile), cut into equal contiguous
// ranges, one per workgroup: a batch of very different lengths keeps every CU
// busy to the end, and the host needs to know no length.  A range covers the
// end of one tile, some whole ones and the start of another; whole ones are
// written out, the cut pieces (at most two a workgroup) leave their sums in
// the workspace for paged_join_kernel.
// Bound by HBM, and by some 10 us before the first keys arrive and for the join.
// bf16, 32 heads over 8 of 128: 64 sequences of up to 8191, 413 MB, 72 us and 4.6
// for the join; one of 131071, 537 MB, 85 and 5.7 (6.3 TB/s while it walks; reads
// alone reach 6.75 here).  Large tiles of wavefronts, more workgroups, or the next
// piece's first keys loaded under this one's merge took as long or longer.

constexpr int PD_UNIT = 32 * PA_WAVES;

// Tiles of a sequence, and units of each; one without keys has one unit, which
// writes its rows.
__device__ __forceinline__ int pd_tiles(const PgSeq& q, int grp) { return (q.n * grp + 15) >> 4; }
__device__ __forceinline__ int pd_units(const PgSeq& q, int unit) {
    return q.kv <= unit ? 1 : (q.kv + unit - 1) / unit;
}

template <class A, bool ONCE>
__global__ __launch_bounds__(64 * PA_WAVES, A::RESIDENT) void paged_rows16_kernel(typename A::Cache c, PagedRows b, int grp, int unit,
                                                                        const typename A::Row* __restrict__ q, int ldq, float scale,
                                                                        typename A::Row* __restrict__ out, int ldo,
                                                                        float* __restrict__ part,
                                                                        PgJoin* __restrict__ joins) {
    using T = typename A::Row;
    constexpr int HD = A::DIM;
    constexpr int NO = 4 * A::VW;
    __shared__ float s_o[PA_WAVES - 1][NO][64];
    __shared__ float s_m[PA_WAVES][16], s_l[PA_WAVES][16];
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const auto units_of = [&](const PgSeq& x) { return pd_tiles(x, grp) * pd_units(x, unit); };
    PgUnits<decltype(units_of)> pu(b, units_of, !b.row_start && b.cap <= unit ? (grp + 15) >> 4 : 0);
    const int units = pu.total, total = units * c.kv_heads, n_wgs = min((int)gridDim.x, total);
    if ((int)blockIdx.x >= n_wgs) {
        if (joins && threadIdx.x == 0) joins[blockIdx.x].rows = 0;
        return;
    }
    const int begin = pg_start(blockIdx.x, total, n_wgs), stop = pg_start(blockIdx.x + 1, total, n_wgs);
    int head = (unsigned)begin / (unsigned)units, u;
    int s = pu.find(begin - head * units, u);
    for (int at = begin; at < stop;) {
        const PgSeq sq = pu.get(s);
        const int all = sq.n * grp, nt = pd_tiles(sq, grp), n = pd_units(sq, unit);
        if (nt == 0) {  // (a sequence without rows)
            u = 0;
            if (++s == b.n_seqs) {
                s = 0;
                head++;
            }
            continue;
        }
        const int tile = u / n, u0 = u - tile * n, m = min(n - u0, stop - at);  // units u0 .. u0 + m - 1 of the tile
        const int i0 = 16 * tile, i = min(i0 + r, all - 1), pos0 = sq.kv - sq.n;
        const int row = sq.row0 + i / grp, h = head * grp + i % grp;
        A a;
        a.load_q(q + (size_t)row * ldq + (size_t)h * HD, scale);
        a.limit = pos0 + i / grp;
        a.start();
        const int first = pos0 + i0 / grp, seen = pos0 + min(i0 + 15, all - 1) / grp + 1;  // keys that some row sees
        const int k0 = u0 * unit, k1 = max(k0, min(seen, (u0 + m) * unit));
        const int per = ((k1 - k0 + A::STEP - 1) / A::STEP + PA_WAVES - 1) / PA_WAVES;
        const int* table = b.table + (size_t)s * b.max_pages;
        const int j0 = k0 + A::STEP * w * per, j1 = min(k1, j0 + A::STEP * per);
        a.template walk<ONCE>(c, table, head, j0, j1, sq.kv, first);
        a.walk_odd(c, table, head, j0, j1, sq.kv, q + (size_t)row * ldq + (size_t)h * HD, scale);
        a.finish();
        if (w > 0) {
#pragma unroll
            for (int t = 0; t < A::VW; t++)
#pragma unroll
                for (int k = 0; k < 4; k++) s_o[w - 1][4 * t + k][lane] = a.o[t][k];
        }
        if (g == 0) {
            s_m[w][r] = a.m;
            s_l[w][r] = a.l;
        }
        __syncthreads();
        const bool whole = m == n;
        if (w == 0 && i0 + r < all) {
            float mx = s_m[0][r], l = 0.0f, wt[PA_WAVES];
#pragma unroll
            for (int v = 1; v < PA_WAVES; v++) mx = fmaxf(mx, s_m[v][r]);
#pragma unroll
            for (int v = 0; v < PA_WAVES; v++) {
                wt[v] = __builtin_amdgcn_exp2f(s_m[v][r] - mx);
                l += s_l[v][r] * wt[v];
            }
            float* slot = part + ((size_t)2 * blockIdx.x + (at != begin)) * pg_slot(16, HD);
            // (of a bad length, or before position 0, all sums are 0)
            const float inv = !whole ? 1.0f : sq.bad ? pg_nan() : a.limit < 0 ? 0.0f : 1.0f / l;
            T* dst = out + (size_t)row * ldo + (size_t)h * HD + 4 * A::VW * g;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                float x[A::VW];
#pragma unroll
                for (int t = 0; t < A::VW; t++) {
                    x[t] = a.o[t][k] * wt[0];
#pragma unroll
                    for (int v = 1; v < PA_WAVES; v++) x[t] = fmaf(s_o[v - 1][4 * t + k][lane], wt[v], x[t]);
                    x[t] *= inv;
                }
                if (whole) {
                    T y[A::VW];
#pragma unroll
                    for (int t = 0; t < A::VW; t++) y[t] = (T)x[t];
                    __builtin_memcpy(__builtin_assume_aligned(dst + A::VW * k, 8), y, sizeof y);
                } else {
                    __builtin_memcpy(__builtin_assume_aligned(slot + r * HD + A::VW * (4 * g + k), 16), x, sizeof x);
                }
            }
            if (!whole && g == 0) {
                slot[16 * HD + r] = mx;
                slot[16 * HD + 16 + r] = l;
            }
        }
        at += m;
        if (at == stop && joins && threadIdx.x == 0)
            joins[blockIdx.x] = pg_join(u0 == 0 && !whole, min(16, all - i0), sq, head, i0, at - m + n - 1, total,
                                        n_wgs, 2 * blockIdx.x + (at - m != begin));
        u += m;
        if (u == nt * n) {
            u = 0;
            if (++s == b.n_seqs) {
                s = 0;
                head++;
            }
        }
        if (at < stop) __syncthreads();  // the merge's LDS is read
    }
}

// Whole tiles of short walks, a wavefront each: where a tile is a few blocks of
// 32 keys, waiting for memory in turn is all that it does, and eight or more of
// them, not two or three, wait on a CU at a time; nor is there a merge.  One
// token a sequence, 128 dims, us, four wavefronts a tile / one:
//   keys          20          60         120         250          500
//    512 tiles  7.7/6.6     8.2/7.6   10.0/12.0   16.1/19.8   25.5/33.7
//    768       11.2/6.2    12.6/8.1   15.9/13.2   22.3/21.9   35.3/38.5
//   4096       46.9/17.2   49.3/25.3  65.6/44.1   98.4/87.9  169.7/169.1
// and up to half as long again where a batch's lengths differ much.
template <class A, bool ONCE>
__global__ __launch_bounds__(64 * PA_WAVES, A::RESIDENT) void paged_rows16_alone_kernel(typename A::Cache c, PagedRows b, int grp, int each,
                                                                              const typename A::Row* __restrict__ q, int ldq, float scale,
                                                                              typename A::Row* __restrict__ out, int ldo) {
    using T = typename A::Row;
    constexpr int HD = A::DIM;
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int at = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * PA_WAVES + (threadIdx.x >> 6)));
    const auto tiles_of = [&](const PgSeq& x) { return pd_tiles(x, grp); };
    PgUnits<decltype(tiles_of)> pu(b, tiles_of, each);
    if (at >= pu.total * c.kv_heads) return;
    const int head = (unsigned)at / (unsigned)pu.total;
    int tile;
    const int s = pu.find(at - head * pu.total, tile);
    const PgSeq sq = pu.get(s);
    const int all = sq.n * grp, i0 = 16 * tile, i = min(i0 + r, all - 1), pos0 = sq.kv - sq.n;
    const int row = sq.row0 + i / grp, h = head * grp + i % grp;
    A a;
    a.load_q(q + (size_t)row * ldq + (size_t)h * HD, scale);
    a.limit = pos0 + i / grp;
    a.start();
    const int* table = b.table + (size_t)s * b.max_pages;
    const int seen = pos0 + min(i0 + 15, all - 1) / grp + 1;  // keys that some row sees
    a.template walk<ONCE>(c, table, head, 0, seen, sq.kv, pos0 + i0 / grp);
    a.walk_odd(c, table, head, 0, seen, sq.kv, q + (size_t)row * ldq + (size_t)h * HD, scale);
    a.finish();
    if (i0 + r >= all) return;
    const float inv = sq.bad ? pg_nan() : a.limit < 0 ? 0.0f : 1.0f / a.l;  // (o is 0 in the first two)
    T* dst = out + (size_t)row * ldo + (size_t)h * HD + 4 * A::VW * g;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        T y[A::VW];
#pragma unroll
        for (int t = 0; t < A::VW; t++) y[t] = (T)(a.o[t][k] * inv);
        __builtin_memcpy(__builtin_assume_aligned(dst + A::VW * k, 8), y, sizeof y);
    }
}

// Sizes of a call of the 16-row kernels: keys a unit, and workgroups (a range
// each, no more than the units that lengths up to cap can have) or, alone, the
// wavefronts of a tile each.  size: bytes of a cached value.
struct Rows16Plan {
    int unit, wgs;
    bool cut, alone;
};
inline Rows16Plan rows16_plan(const PagedKv& kv, const PagedRows& r, int n_heads, int hd, int size) {
    const int grp = n_heads / kv.kv_heads;
    const long tiles = pg_tiles_bound(r, grp, 16) * kv.kv_heads;
    Rows16Plan p;
    p.unit = pg_whole(kv, r, n_heads, hd) ? PG_WHOLE_KEYS : PD_UNIT;
    const long units = tiles * (r.cap > p.unit ? ((long)r.cap + p.unit - 1) / p.unit : 1);
    p.cut = r.cap > p.unit;
    const int most = PG_WGS / 2 * pg_resident(hd, size);
    p.wgs = (int)(units < most || !p.cut ? units : most);
    p.alone = r.cap <= 32 || (r.cap <= 256 && tiles > PG_WGS);
    return p;
}

inline size_t rows16_work_bytes(const PagedKv& kv, const PagedRows& r, int n_heads, int hd, int size) {
    const Rows16Plan p = rows16_plan(kv, r, n_heads, hd, size);
    return p.cut ? p.wgs * (2 * pg_slot(16, hd) * sizeof(float) + sizeof(PgJoin)) : 0;
}

inline bool rows16_fits(const PagedKv& kv, const PagedRows& r, int n_heads, int hd, int size) {
    const long tiles = pg_tiles_bound(r, n_heads / kv.kv_heads, 16) * kv.kv_heads;
    if (tiles > 0x7fffffff / (r.cap / PD_UNIT + 1)) return false;
    const Rows16Plan p = rows16_plan(kv, r, n_heads, hd, size);
    return p.wgs <= (p.alone ? PA_WAVES * PG_GRID : PG_GRID);
}

template <class A>
hipError_t rows16_launch(const PagedAttendArgs& p, const typename A::Cache& c, hipStream_t s) {
    using T = typename A::Row;
    const int grp = p.n_heads / c.kv_heads;
    const Rows16Plan pl = rows16_plan(c, p.rows, p.n_heads, A::DIM, A::BYTES / A::DIM);
    float* part = static_cast<float*>(p.work);
    PgJoin* joins = pl.cut ? reinterpret_cast<PgJoin*>(part + (size_t)2 * pl.wgs * pg_slot(16, A::DIM)) : nullptr;
    // Past the caches where one tile reads its keys alone and the batch's may
    // exceed the 256 MB last-level cache (537 MB 103.9 -> 92.8 us, 201 MB 55.6
    // -> 50.5; what the cache still holds of 82 MB it would lose, 26.8 -> 29.1)
    const double bytes = (double)p.rows.n_seqs * p.rows.cap * c.kv_heads * A::BYTES * 2;
    const bool once = !p.rows.row_start && grp <= 16 && bytes > 256e6;
    if (pl.alone) {
        const auto kernel = once ? paged_rows16_alone_kernel<A, true> : paged_rows16_alone_kernel<A, false>;
        hipLaunchKernelGGL(kernel, dim3((pl.wgs + PA_WAVES - 1) / PA_WAVES), dim3(64 * PA_WAVES), 0, s, c, p.rows, grp,
                           p.rows.row_start ? 0 : (grp + 15) >> 4, static_cast<const T*>(p.q), p.ldq, p.scale,
                           static_cast<T*>(p.out), p.ldo);
        return hipGetLastError();
    }
    const auto kernel = once ? paged_rows16_kernel<A, true> : paged_rows16_kernel<A, false>;
    hipLaunchKernelGGL(kernel, dim3(pl.wgs), dim3(64 * PA_WAVES), 0, s, c, p.rows, grp, pl.unit,
                       static_cast<const T*>(p.q), p.ldq, p.scale, static_cast<T*>(p.out), p.ldo, part, joins);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || !pl.cut) return e;
    return launch_paged_join(pg_dtype<T>(), A::DIM, joins, part, pl.wgs, pg_tiles_bound(p.rows, grp, 16) * c.kv_heads,
                             16, p.rows.row_start || grp > 16 ? 16 : grp, grp, false, p.out, p.ldo, s);
}

}  // namespace frq
