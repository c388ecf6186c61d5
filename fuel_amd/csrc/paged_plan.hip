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

constexpr int PP_WG = 1024;
constexpr int PP_WAVES = PP_WG / 64;

// Sums of v >= 0 over threads 0 .. the own one; their total in `all`.  `s` is free
// again behind the next barrier but one.
__device__ __forceinline__ int pp_scan(int v, int (&s)[PP_WAVES], int& all) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, sum = pg_scan(v);
    __syncthreads();
    if (lane == 63) s[w] = sum;
    __syncthreads();
    const int part = pg_scan(lane < PP_WAVES ? s[lane] : 0);
    all = __builtin_amdgcn_readlane(part, PP_WAVES - 1);
    return pg_add(sum, w ? __builtin_amdgcn_readlane(part, w - 1) : 0);
}

// The first of n threads whose sum is past i.
__device__ __forceinline__ int pp_find(const int (&sums)[PP_WG], int i) {
    int lo = 0;
#pragma unroll
    for (int step = PP_WG / 2; step; step /= 2)
        if (sums[lo + step - 1] <= i) lo += step;
    return lo;
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

__global__ __launch_bounds__(PP_WG) void paged_plan_kernel(PagedPlanArgs a) {
    __shared__ int s_wave[PP_WAVES], s_sum[PP_WG], s_first[PP_WG];
    const int tid = threadIdx.x, ps1 = (1 << a.log_ps) - 1;
    const auto pages = [&](int n) { return (int)(((unsigned)n + ps1) >> a.log_ps); };
    int stack = min(max(*a.n_free, 0), a.n_pages);
    // drops
    for (int base = 0; base < a.n_seqs; base += PP_WG) {
        const PpSeq q = pp_seq(a, base + tid);
        const int keep = q.tokens < 0 ? pages(max(q.kv + q.tokens, 0)) : 0, n = q.tokens < 0 ? pages(q.kv) - keep : 0;
        int all;
        const int sum = pp_scan(n, s_wave, all);
        if (all == 0) continue;
        s_sum[tid] = sum;
        s_first[tid] = keep - (sum - n);
        __syncthreads();
        all = min(all, a.n_pages - stack);  // (lengths of more pages than there are)
        for (int i = tid; i < all; i += PP_WG) {
            const int t = pp_find(s_sum, i);
            a.free_pages[stack + i] = a.table[(size_t)(base + t) * a.max_pages + s_first[t] + i];
        }
        stack += all;
    }
    __syncthreads();
    // grants
    int asked_pages = 0, asked_rows = 0, rows = 0, taken = 0;
    for (int base = 0; base < a.n_seqs; base += PP_WG) {
        const int s = base + tid;
        const PpSeq q = pp_seq(a, s);
        const int want = max(q.tokens, 0), have = q.tokens > 0 ? pages(q.kv) : 0;
        const int need = q.tokens > 0 ? pages(q.kv + want) - have : 0;
        int all_pages, all_rows, all_granted, all_taken;
        const int sum_pages = pg_add(asked_pages, pp_scan(need, s_wave, all_pages));
        const int sum_rows = pg_add(asked_rows, pp_scan(want, s_wave, all_rows));
        const bool ok = want > 0 && (need == 0 || sum_pages <= stack) && sum_rows <= a.rows;
        const int granted = ok ? want : 0, sum = pp_scan(granted, s_wave, all_granted);
        const int mine = pp_scan(ok ? need : 0, s_wave, all_taken);
        s_sum[tid] = mine;
        s_first[tid] = have - (mine - (ok ? need : 0));
        if (s < a.n_seqs) {
            a.kv_len_out[s] = q.tokens < 0 ? max(q.kv + q.tokens, 0) : q.kv + granted;
            a.row_start[s] = rows + sum - granted;
        }
        __syncthreads();
        for (int i = tid; i < all_taken; i += PP_WG) {
            const int t = pp_find(s_sum, i);
            a.table[(size_t)(base + t) * a.max_pages + s_first[t] + i] = a.free_pages[stack - 1 - taken - i];
        }
        asked_pages = pg_add(asked_pages, all_pages);
        asked_rows = pg_add(asked_rows, all_rows);
        rows += all_granted;
        taken += all_taken;
    }
    if (tid == 0) {
        a.row_start[a.n_seqs] = rows;
        *a.n_free_out = stack - taken;
    }
}

// Slot and position of each packed row, -1 behind the last.
__global__ __launch_bounds__(256) void paged_slots_kernel(PagedPlanArgs a) {
    const int row = blockIdx.x * 256 + threadIdx.x;
    if (row >= a.rows) return;
    int64_t slot = -1;
    int pos = -1;
    if (row < a.row_start[a.n_seqs]) {
        int lo = 0, n = a.n_seqs;  // the last of lo .. lo + n - 1 that starts at or before row
        while (n > 1) {
            const int half = n >> 1;
            if (a.row_start[lo + half] <= row) {
                lo += half;
                n -= half;
            } else {
                n = half;
            }
        }
        pos = a.kv_len_out[lo] - (a.row_start[lo + 1] - row);
        const int page = a.table[(size_t)lo * a.max_pages + (pos >> a.log_ps)];
        slot = ((int64_t)page << a.log_ps) + (pos & ((1 << a.log_ps) - 1));
    }
    if (a.slots) a.slots[row] = slot;
    if (a.positions) a.positions[row] = pos;
}

}  // namespace

hipError_t launch_paged_plan(const PagedPlanArgs& p, hipStream_t s) {
    hipLaunchKernelGGL(paged_plan_kernel, dim3(1), dim3(PP_WG), 0, s, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.rows == 0 || !(p.slots || p.positions)) return e;
    hipLaunchKernelGGL(paged_slots_kernel, dim3((unsigned)((p.rows + 255l) / 256)), dim3(256), 0, s, p);
    return hipGetLastError();
}

}  // namespace frq
