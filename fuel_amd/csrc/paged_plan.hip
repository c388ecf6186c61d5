// Pages of a pool for the sequences of a batch: what paged.hpp's batches consist of,
// built where they are read, so that a captured step needs no host.
//
// A sequence of length n with t tokens asked for holds pages ceil(n / ps) ..
// ceil((n + t) / ps) - 1 more.  The pool's free pages are a stack; in sequence order
//   t < 0   the last -t tokens are dropped, the pages past the new end pushed
//   t > 0   granted if the pages asked for so far fit the stack (or it asks for none)
//           and the tokens asked for so far fit the rows: both are sums over the
//           sequences before it, granted or not, so that a request that does not fit
//           is not overtaken by later ones for pages
// all drops before all grants.  Three scans over the sequences, in one workgroup:
// latency, nothing else.  Sums saturate at 2^31 - 1, which no stack and no rows hold.
#include <hip/hip_runtime.h>

#include "common.hpp"
#include "kernels.hpp"
#include "paged.hpp"

namespace frq {

namespace {

// Rows a thread whose slots the one workgroup writes itself: a second launch costs
// more than they do (256 sequences of one token each 7.4 us with it, 6.3 without).
constexpr int PP_ROWS = 4;

// Sums of N values >= 0 each over the threads before (in place), totals in `all`.
// `s` is free again behind the next barrier but one.
template <int N, int WAVES>
__device__ __forceinline__ void pp_scan(int (&v)[N], int (&s)[2][WAVES], int (&all)[N]) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
    for (int k = 0; k < N; k++) v[k] = pg_scan(v[k]);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; k++)
        if (lane == 63) s[k][w] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; k++) {
        const int part = pg_scan(lane < WAVES ? s[k][lane] : 0), before = __shfl_up(v[k], 1);
        all[k] = __builtin_amdgcn_readlane(part, 63);
        v[k] = pg_add(lane ? before : 0, w ? __builtin_amdgcn_readlane(part, w - 1) : 0);
    }
}

// The first of N (a power of two) whose sum is past i, which the last one's is.
template <int N>
__device__ __forceinline__ int pp_find(const int (&sums)[N], int i) {
    int lo = 0;
#pragma unroll
    for (int step = N / 2; step; step /= 2)
        if (sums[lo + step - 1] <= i) lo += step;
    return lo;
}

// store(t, i, load(t, i)) of each of `count` items i, t the one of N whose sum holds it.
// Four items a thread at a time where there are that many: their searches and loads
// do not wait for each other.
template <int WG, int N, class Load, class Store>
__device__ __forceinline__ void pp_each(const int (&sums)[N], int count, Load load, Store store) {
    if (count <= WG) {
        const int i = threadIdx.x;
        if (i < count) {
            const int t = pp_find(sums, i);
            store(t, i, load(t, i));
        }
        return;
    }
    for (int i = threadIdx.x; i < count; i += 4 * WG) {
        int t[4], v[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int x = min(i + u * WG, count - 1);
            t[u] = pp_find(sums, x);
            v[u] = load(t[u], x);
        }
#pragma unroll
        for (int u = 0; u < 4; u++)
            if (i + u * WG < count) store(t[u], i + u * WG, v[u]);
    }
}

struct PpSeq {
    int kv, tokens;
};
__device__ __forceinline__ PpSeq pp_seq(const PagedPlanArgs& a, int s) {
    PpSeq q{0, 0};
    if (s < a.n_seqs) {
        q.kv = a.kv_len[s];
        q.tokens = a.tokens[s];
        const int cap = a.max_pages << a.log_ps;
        // (no length: it stays; more than the table holds: not granted)
        if (q.kv < 0 || q.kv > cap || q.tokens > cap - q.kv) q.tokens = 0;
    }
    return q;
}

// Slot and position of a row at position pos (-1: none) in a page.
__device__ __forceinline__ void pp_slot(const PagedPlanArgs& a, int row, int pos, int page) {
    if (a.slots) a.slots[row] = pos < 0 ? -1 : ((int64_t)page << a.log_ps) + (pos & ((1 << a.log_ps) - 1));
    if (a.positions) a.positions[row] = pos;
}

// One workgroup of WG threads, a thread K sequences at a time.
template <int K, int WG>
__global__ __launch_bounds__(WG) void paged_plan_kernel(PagedPlanArgs a) {
    constexpr int n = K * WG;
    __shared__ int s_wave[2][WG / 64], s_sum[n], s_first[n];
    const int tid = threadIdx.x, ps1 = (1 << a.log_ps) - 1;
    const auto pages = [&](int x) { return (int)(((unsigned)x + ps1) >> a.log_ps); };
    PpSeq q[K];
#pragma unroll
    for (int k = 0; k < K; k++) q[k] = pp_seq(a, K * tid + k);
    int stack = min(max(*a.n_free, 0), a.n_pages);
    // drops
    for (int base = 0; base < a.n_seqs; base += n) {
        int keep[K], gone[K], sum[1] = {0}, all[1];
#pragma unroll
        for (int k = 0; k < K; k++) {
            if (base) q[k] = pp_seq(a, base + K * tid + k);
            keep[k] = pages(max(q[k].kv + min(q[k].tokens, 0), 0));
            gone[k] = q[k].tokens < 0 ? pages(q[k].kv) - keep[k] : 0;
            sum[0] = pg_add(sum[0], gone[k]);
        }
        if (!__syncthreads_or(sum[0])) continue;
        pp_scan(sum, s_wave, all);
        int at = sum[0];
#pragma unroll
        for (int k = 0; k < K; k++) {
            s_first[K * tid + k] = keep[k] - at;
            at = pg_add(at, gone[k]);
            s_sum[K * tid + k] = at;
        }
        __syncthreads();
        const int put = min(all[0], a.n_pages - stack);  // (lengths of more pages than there are)
        pp_each<WG>(
            s_sum, put, [&](int t, int i) { return a.table[(size_t)(base + t) * a.max_pages + s_first[t] + i]; },
            [&](int, int i, int page) { a.free_pages[stack + i] = page; });
        stack += put;
    }
    __syncthreads();
    // grants
    const bool slots = a.rows <= PP_ROWS * WG && (a.slots || a.positions);
    int asked_pages = 0, asked_rows = 0, rows = 0, taken = 0;
    for (int base = 0; base < a.n_seqs; base += n) {
        int want[K], have[K], need[K], sum[2] = {0, 0}, all[2];
#pragma unroll
        for (int k = 0; k < K; k++) {
            if (a.n_seqs > n) q[k] = pp_seq(a, base + K * tid + k);
            want[k] = max(q[k].tokens, 0);
            have[k] = pages(q[k].kv);
            need[k] = want[k] ? pages(q[k].kv + want[k]) - have[k] : 0;
            sum[0] = pg_add(sum[0], need[k]);
            sum[1] = pg_add(sum[1], want[k]);
        }
        pp_scan(sum, s_wave, all);
        const int end_pages = pg_add(asked_pages, all[0]), end_rows = pg_add(asked_rows, all[1]);
        if (end_pages > stack || end_rows > a.rows) {  // not all: the sums of those that are
            int at_pages = pg_add(asked_pages, sum[0]), at_rows = pg_add(asked_rows, sum[1]);
            sum[0] = sum[1] = 0;
#pragma unroll
            for (int k = 0; k < K; k++) {
                at_pages = pg_add(at_pages, need[k]);
                at_rows = pg_add(at_rows, want[k]);
                if ((need[k] && at_pages > stack) || at_rows > a.rows) want[k] = need[k] = 0;
                sum[0] += need[k];
                sum[1] += want[k];
            }
            pp_scan(sum, s_wave, all);
        }
        asked_pages = end_pages;
        asked_rows = end_rows;
        int at = sum[0], row = sum[1];
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int s = base + K * tid + k;
            s_first[K * tid + k] = have[k] - at;
            at += need[k];
            s_sum[K * tid + k] = at;
            if (s < a.n_seqs) {
                a.kv_len_out[s] = q[k].tokens < 0 ? max(q[k].kv + q[k].tokens, 0) : q[k].kv + want[k];
                a.row_start[s] = rows + row;
            }
            row += want[k];
        }
        __syncthreads();
        pp_each<WG>(
            s_sum, all[0], [&](int, int i) { return a.free_pages[stack - 1 - taken - i]; },
            [&](int t, int i, int page) { a.table[(size_t)(base + t) * a.max_pages + s_first[t] + i] = page; });
        if (slots) {
            __syncthreads();
            row = sum[1];
#pragma unroll
            for (int k = 0; k < K; k++) {
                s_first[K * tid + k] = q[k].kv - row;  // position of the sequence's row i: that and i
                row += want[k];
                s_sum[K * tid + k] = row;
            }
            __syncthreads();
            pp_each<WG>(
                s_sum, all[1],
                [&](int t, int i) {
                    return a.table[(size_t)(base + t) * a.max_pages + ((s_first[t] + i) >> a.log_ps)];
                },
                [&](int t, int i, int page) { pp_slot(a, rows + i, s_first[t] + i, page); });
        }
        rows += all[1];
        taken += all[0];
    }
    if (slots)
        for (int row = rows + tid; row < a.rows; row += WG) pp_slot(a, row, -1, 0);
    if (tid == 0) {
        a.row_start[a.n_seqs] = rows;
        *a.n_free_out = stack - taken;
    }
}

// Slots of more rows, a thread each.
__global__ __launch_bounds__(256) void paged_slots_kernel(PagedPlanArgs a) {
    const int row = blockIdx.x * 256 + threadIdx.x;
    if (row >= a.rows) return;
    if (row >= a.row_start[a.n_seqs]) {
        pp_slot(a, row, -1, 0);
        return;
    }
    int s = 0, n = a.n_seqs;  // the last of s .. s + n - 1 that starts at or before row
    while (n > 1) {
        const int half = n >> 1;
        const bool up = a.row_start[s + half] <= row;
        s += up ? half : 0;
        n = up ? n - half : half;
    }
    const int pos = a.kv_len_out[s] - (a.row_start[s + 1] - row);
    pp_slot(a, row, pos, a.table[(size_t)s * a.max_pages + (pos >> a.log_ps)]);
}

}  // namespace

hipError_t launch_paged_plan(const PagedPlanArgs& p, hipStream_t s) {
    // (few wavefronts meet at a barrier sooner; many move more pages at a time)
    const long most = p.n_seqs > p.rows >> p.log_ps ? p.n_seqs : p.rows >> p.log_ps;
    const int wg = most <= 64 ? 64 : most <= 256 ? 256 : 1024;
    const auto kernel = wg == 64    ? paged_plan_kernel<1, 64>
                        : wg == 256 ? paged_plan_kernel<1, 256>
                        : p.n_seqs <= 1024 ? paged_plan_kernel<1, 1024> : paged_plan_kernel<4, 1024>;
    hipLaunchKernelGGL(kernel, dim3(1), dim3(wg), 0, s, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.rows <= PP_ROWS * wg || !(p.slots || p.positions)) return e;
    hipLaunchKernelGGL(paged_slots_kernel, dim3((unsigned)((p.rows + 255l) / 256)), dim3(256), 0, s, p);
    return hipGetLastError();
}

}  // namespace frq
