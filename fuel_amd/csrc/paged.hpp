// The paged KV cache: argument views and the device helpers its kernels share
// (paged.hip, paged_prefill.hip).
//
// Cache: k and v are [n_pages][kv_heads][page_size][HD] f16 or bf16, so the
// rows of one head in one page are contiguous (16 rows of 128 are 4 KiB).
// Sequence s keeps position j in page table[s * max_pages + j / page_size],
// row j % page_size.  page_size is a power of two >= 16: 16 keys from a
// multiple of 16 never cross a page.
//
// Packed rows: row_start[s] .. row_start[s + 1] - 1 are sequence s's (row s
// alone without a row_start); the last of them stands at position
// kv_len[s] - 1, the ones before it at the positions before.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "common.hpp"

namespace frq {

struct PagedKv {
    void* k;
    void* v;
    int n_pages;
    int log_ps;
    int kv_heads;
};

struct PagedRows {
    const int* table;
    const int* kv_len;
    const int* row_start;  // null: one row a sequence
    int n_seqs;
    int max_pages;
    int rows;
    int cap;  // kv_len beyond it is no length (<= max_pages * page_size)
};

// A bound on the tiles of tile_rows query rows that a batch's sequences have:
// each one's last may be partly empty.
inline long pg_tiles_bound(const PagedRows& r, int grp, int tile_rows) {
    return r.row_start ? (long)r.rows * grp / tile_rows + r.n_seqs
                       : (long)r.n_seqs * ((grp + tile_rows - 1) / tile_rows);
}

// Which kernel a call takes.  ROWS16: 16 query rows a tile, the keys of a call
// over all workgroups (paged.hip).  TILES: 128 rows a tile, a workgroup each;
// CUT: the same, the keys over all workgroups (paged_prefill.hip).  One row a
// sequence: always ROWS16.  Otherwise by what they took, in us, over 1 .. 48
// sequences, 2 .. 3000 new rows after 0 .. 32000 cached, 1 .. 32 KV heads, all
// types (K: keys of the longest sequence, n: tiles times KV heads; the estimate is
// the same for all types, since the workspace's size is):
//   ROWS16  12 + n16 K / 20000        (8 + .. where its tiles stay whole)
//   TILES   10 + 0.034 K max(1/2, n128 / 512)
//   CUT     26 + n128 K / 15000       (the second launch and the pieces' bytes)
// Over 420 such batches the choice is 1.6 % slower than the fastest of the three in
// the mean, at worst by half (the host knows the rows of a batch and its longest
// sequence, not how they go together).  Of 32 heads over 8, bf16: 128 rows after
// 600: 22 / 18 / 27 (ROWS16 / TILES / CUT), 300 after 600: 41 / 20 / 35, 300 after
// 4096: 155 / 64 / 52, 1500 after 600: 248 / 55 / 79.
enum PagedKind { PG_ROWS16, PG_TILES, PG_CUT };
// Whether ROWS16 leaves its tiles whole: short walks, which a second launch
// would cost more than they take.  One token a sequence, cut / whole, us: 8
// tiles of 200 keys of 128 10.6 / 8.2, of 400 10.3 / 10.6, 128 tiles of 400
// 13.2 / 11.4, of 1000 19.6 / 19.9; 8 tiles of 400 keys of 64 9.9 / 7.8.  (Of
// longer ones whole tiles gain up to 10 % where all are as long as the longest
// and there is one for every CU, and lose more where they are not.)
constexpr int PG_WHOLE_KEYS = 1024;
inline bool pg_whole(const PagedKv& kv, const PagedRows& r, int n_heads, int hd) {
    const long tiles = pg_tiles_bound(r, n_heads / kv.kv_heads, 16) * kv.kv_heads;
    return (long)r.cap * hd <= (tiles >= 128 ? 65536 : 32768);
}
inline PagedKind pg_kind(const PagedKv& kv, const PagedRows& r, int n_heads, int hd) {
    if (!r.row_start) return PG_ROWS16;
    const int grp = n_heads / kv.kv_heads;
    const double k = r.cap, n16 = (double)pg_tiles_bound(r, grp, 16) * kv.kv_heads,
                 n128 = (double)pg_tiles_bound(r, grp, 128) * kv.kv_heads;
    const double rows16 = (pg_whole(kv, r, n_heads, hd) ? 8 : 12) + n16 * k / 20000;
    const double tiles = 10 + 0.034 * k * (n128 > 256 ? n128 / 512 : 0.5);
    const double cut = r.cap <= 1 << 24 && n128 <= 4096 ? 26 + n128 * k / 15000 : 1e30;  // (its units are an int)
    if (rows16 <= tiles && rows16 <= cut) return PG_ROWS16;
    return tiles <= cut ? PG_TILES : PG_CUT;
}

// Workgroups of a call whose keys are cut into equal ranges: two a CU, all
// resident at once.
constexpr int PG_WGS = 512;

// Workgroups of 256 threads that one launch can have: HIP's grids end below 2^32
// threads.
constexpr long PG_GRID = (1L << 24) - 1;

// Cut tiles.  Workgroups that share the keys of a tile of `rows` query rows
// leave slots of floats in the workspace, two a workgroup: o [rows][hd]
// (unnormalized), m [rows], l [rows]; and each a record of what is to be joined.
constexpr size_t pg_slot(int rows, int hd) { return (size_t)rows * hd + 2 * rows; }
struct PgJoin {
    int rows;        // of the tile that begins in the workgroup's range and goes on past it; 0: none
    int last, slot;  // workgroup of the tile's last piece; slot of its first
    int row0, pos0;  // the sequence's first packed row, and its position
    int head, i0;    // KV head, the tile's first query row
    int pad;
};

#ifdef __HIPCC__

typedef float pg_f4 __attribute__((ext_vector_type(4)));
typedef uint32_t pg_u4 __attribute__((ext_vector_type(4)));

// Vector types, conversions and MFMAs of a cache element type.
template <class E>
struct PgElem;
template <>
struct PgElem<_Float16> {
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    typedef _Float16 v2 __attribute__((ext_vector_type(2)));
    static constexpr int SPLIT = 2;  // parts that hold an f32 to 2^-22
    static constexpr uint32_t INF = 0x7c007c00u;  // exponent bits of both halves of a word
    // Weights are 2^TOP at most: here as many of their digits as f16's range holds
    // (its largest is 65504).
    static constexpr float TOP = 15.0f;
    __device__ static pg_f4 mfma16(v8 a, v8 b, pg_f4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};
template <>
struct PgElem<__bf16> {
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    typedef __bf16 v2 __attribute__((ext_vector_type(2)));
    static constexpr int SPLIT = 3;  // 8 significant bits each: an f32 to 2^-24
    static constexpr uint32_t INF = 0x7f807f80u;
    // 2^30 keys' weights times values up to f32's largest sum within f32's range.
    static constexpr float TOP = -31.0f;
    __device__ static pg_f4 mfma16(v8 a, v8 b, pg_f4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
};

__device__ __forceinline__ float pg_nan() { return __builtin_nanf(""); }

// A sequence as the kernels see it.  n = 0 where row_start is no range of
// rows; bad where kv_len is no length (its rows' results are NaN).
struct PgSeq {
    int row0, n, kv;
    bool bad;
};
__host__ __device__ __forceinline__ PgSeq pg_seq(const PagedRows& b, int s) {
    PgSeq q;
    q.row0 = s;
    q.n = 1;
    if (b.row_start) {
        q.row0 = b.row_start[s];
        const int end = b.row_start[s + 1];
        q.n = q.row0 >= 0 && end <= b.rows && end > q.row0 ? end - q.row0 : 0;
    }
    q.kv = b.kv_len[s];
    q.bad = q.kv < 0 || q.kv > b.cap;
    if (q.bad) q.kv = 0;
    return q;
}

// The page of position j of a sequence of kv (0 behind its end), and whether it
// is none of the pool's: then its keys are read from page 0 and count as NaN.
__host__ __device__ __forceinline__ int pg_page(const PagedKv& c, const int* table, int j, int kv, bool& none) {
    const int id = j < kv ? table[j >> c.log_ps] : 0;
    none = (unsigned)id >= (unsigned)c.n_pages;
    return none ? 0 : id;
}

// Maximum of no scores: below every finite one, and finite itself, so that a row
// that has seen nothing keeps weights, sums and factors that are numbers.
constexpr float PG_LEAST = -__FLT_MAX__;

// f16 parts hold weights in steps of 2^-24.  Where keys have weights far below the
// largest so far, the score that stands for the weight 1 follows theirs down, so
// that those weights keep their digits too, by up to 2^PG_DROP: the sums stay in
// f32's range (2^15 a weight, 2^16 a value, 2^30 keys), and what is lost is below
// 2^-PG_DROP of what f32 sums keep.
constexpr float PG_DROP = 40.0f;

// Whether an infinite or NaN value is among a lane's sums.
template <int N, class V>
__device__ __forceinline__ bool pg_odd(const V (&o)[N]) {
    float t = 0.0f;
#pragma unroll
    for (int n = 0; n < N; n++)
#pragma unroll
        for (int i = 0; i < (int)(sizeof(V) / sizeof(float)); i++) t = fmaf(o[n][i], 0.0f, t);
    return t != t;
}

// Whether all of them are NaN: nothing more changes them.
template <int N, class V>
__device__ __forceinline__ bool pg_all_nan(const V (&o)[N]) {
    bool all = true;
#pragma unroll
    for (int n = 0; n < N; n++)
#pragma unroll
        for (int i = 0; i < (int)(sizeof(V) / sizeof(float)); i++) all &= o[n][i] != o[n][i];
    return all;
}

// Whether a word holds an infinite or NaN half.
template <class E>
__device__ __forceinline__ bool pg_word_odd(uint32_t w) {
    const uint32_t t = ~w & PgElem<E>::INF;
    return (t & 0xffffu) == 0 || (t >> 16) == 0;
}

// Adds keys j0 .. j1 - 1 to a row's maximum and sums as the definition has them:
// f32 dot products, whole weights, no key that the row does not see.  The kernels'
// products form q and the weights in parts, and of a tile's rows some see keys that
// others do not: 0 * inf, and inf in parts of both signs, are NaN there where the
// definition has a number or an infinity.  Such sums never become finite again, so
// keys that end with one are walked a second time, and the blocks of them that hold
// an infinite or NaN value come here.  SHARE lanes, 64 / SHARE apart, hold a row of
// HD dims; a lane's are RUNS runs of 4, run i from dim(i) on.  x: the row's q (from
// memory: in the registers there is room for the kernels' own loops only); own_l:
// whether l is the lane's; a weight is 2^shift at most; add(i, e, f, p, v): sum e of
// run i becomes f times itself and p v.
template <class E, class T, int HD, int SHARE, class Dim, class Add>
__device__ __forceinline__ void pg_plain(const PagedKv& c, const int* table, int head, const T* x, float scale,
                                         int limit, int j0, int j1, float shift, bool own_l, Dim dim, Add add,
                                         float& m, float& l) {
    constexpr int RUNS = HD / SHARE / 4, KEYS = 4;  // keys at a time: q is read once for them
    const float factor = scale * 1.4426950408889634f;
#pragma unroll 1
    for (int j = j0; j < j1; j += KEYS) {  // (of one page: j0 is a multiple of 16)
        bool none;
        const int page = pg_page(c, table, j, j + 1, none);
        const size_t row = ((((size_t)page * c.kv_heads + head) << c.log_ps) + (j & ((1 << c.log_ps) - 1))) * HD;
        const E *k = static_cast<const E*>(c.k) + row, *v = static_cast<const E*>(c.v) + row;
        float s[KEYS] = {}, mn = m;
#pragma unroll 2
        for (int i = 0; i < RUNS; i++) {
            T z[4];
            __builtin_memcpy(z, __builtin_assume_aligned(x + dim(i), 8), sizeof z);
#pragma unroll
            for (int u = 0; u < KEYS; u++) {
                E y[4];
                __builtin_memcpy(y, __builtin_assume_aligned(k + u * HD + dim(i), 8), sizeof y);
#pragma unroll
                for (int e = 0; e < 4; e++) s[u] = fmaf((float)z[e] * factor, (float)y[e], s[u]);
            }
        }
#pragma unroll
        for (int u = 0; u < KEYS; u++) {
#pragma unroll
            for (int d = 64 / SHARE; d < 64; d *= 2) s[u] += __shfl_xor(s[u], d);
            if (none) s[u] = pg_nan();
            if (j + u <= limit) mn = fmaxf(mn, s[u]);
        }
        if (j > limit) continue;
        const float f = __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        l *= f;
#pragma unroll
        for (int u = 0; u < KEYS; u++) {
            if (j + u > limit) break;
            const float p = __builtin_amdgcn_exp2f(s[u] - mn + shift);
            if (own_l) l += p;
#pragma unroll
            for (int i = 0; i < RUNS; i++) {
                E y[4];
                __builtin_memcpy(y, __builtin_assume_aligned(v + u * HD + dim(i), 8), sizeof y);
#pragma unroll
                for (int e = 0; e < 4; e++) add(i, e, u ? 1.0f : f, p, (float)y[e]);
                if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // (few loads at once: the sums fill the registers)
            }
        }
    }
}

// Sums of v >= 0 over lanes 0 .. the own one, at most 0x7fffffff, by DPP (a chain
// of lane shuffles takes ten times as long).
__device__ __forceinline__ int pg_add(int a, int b) { return __builtin_elementwise_add_sat(a, b); }
__device__ __forceinline__ int pg_scan(int v) {
#define FRQ_DPP_ADD(ctrl, rmask) v = pg_add(v, __builtin_amdgcn_update_dpp(0, v, ctrl, rmask, 0xF, false))
    FRQ_DPP_ADD(0x111, 0xF);  // row_shr 1, 2, 4, 8: sums within each 16-lane row
    FRQ_DPP_ADD(0x112, 0xF);
    FRQ_DPP_ADD(0x114, 0xF);
    FRQ_DPP_ADD(0x118, 0xF);
    FRQ_DPP_ADD(0x142, 0xA);  // row_bcast:15 -> rows 1, 3 add the row before
    FRQ_DPP_ADD(0x143, 0xC);  // row_bcast:31 -> rows 2, 3 add rows 0 + 1
#undef FRQ_DPP_ADD
    return v;
}

// Where the units of a batch's sequences lie, units(PgSeq) >= 0 of them one
// sequence after another, and 64 of its sequences in a wavefront's registers.
// Every lane takes part, results are wave-uniform.  Lane l adds up the
// sequences [l share, (l + 1) share), whose loads do not wait for each other;
// a lookup then loads one share: two memory round trips for any n_seqs <= 4096.
// each: every sequence has so many units (0: not known), and none is loaded
// before the lookup.  A batch whose sequences have more rows together than it has
// (row_start lists rows over and over) has no units: its tiles can be more than
// pg_tiles_bound(), and a grid of that would drop some, of any sequence.
template <class F>
struct PgUnits {
    const PagedRows& b;
    F units;
    PgSeq own;  // lane l: sequence s0 + l
    int s0, share, sum, total, each;

    __device__ __forceinline__ void load(int base) {
        const int s = base + (int)(threadIdx.x & 63);
        s0 = base;
        own = PgSeq{0, 0, 0, false};
        if (s < b.n_seqs) own = pg_seq(b, s);
    }
    __device__ __forceinline__ int mine() const { return s0 + (int)(threadIdx.x & 63) < b.n_seqs ? units(own) : 0; }
    __device__ __forceinline__ PgUnits(const PagedRows& rows, F f, int each_ = 0)
        : b(rows), units(f), each(each_) {
        share = (b.n_seqs + 63) >> 6;
        if (each) {
            s0 = -64;
            total = b.n_seqs * each;
            return;
        }
        int v = 0, n = 0;
        if (share == 1) {
            load(0);
            v = mine();
            n = own.n;
        } else {
            s0 = -64;
            const int from = share * (int)(threadIdx.x & 63), to = min(b.n_seqs, from + share);
#pragma unroll 4
            for (int s = from; s < to; s++) {
                const PgSeq q = pg_seq(b, s);
                v = pg_add(v, units(q));
                n = pg_add(n, q.n);
            }
        }
        sum = pg_scan(v);
        total = __builtin_amdgcn_readlane(sum, 63);
        if (b.row_start && __builtin_amdgcn_readlane(pg_scan(n), 63) > b.rows) total = 0;
    }
    // The sequence that holds unit at < total, and the unit's number in it.
    __device__ __forceinline__ int find(int at, int& in_seq) {
        if (each) {
            const int s = (unsigned)at / (unsigned)each;
            in_seq = at - s * each;
            return s;
        }
        int l = __builtin_ctzll(__ballot(sum > at)), base = l * share;
        if (share == 1) {
            in_seq = at - (l ? __builtin_amdgcn_readlane(sum, l - 1) : 0);
            return l;
        }
        at -= l ? __builtin_amdgcn_readlane(sum, l - 1) : 0;
        for (;; base += 64) {
            load(base);
            const int u = mine(), v = pg_scan(u);
            const uint64_t past = __ballot(v > at);
            if (past) {
                l = __builtin_ctzll(past);
                in_seq = at - __builtin_amdgcn_readlane(v - u, l);
                return base + l;
            }
            at -= __builtin_amdgcn_readlane(v, 63);
        }
    }
    // Sequence s < n_seqs.
    __device__ __forceinline__ PgSeq get(int s) {
        if (s < s0 || s >= s0 + 64) load(s);
        const int l = s - s0;
        return PgSeq{__builtin_amdgcn_readlane(own.row0, l), __builtin_amdgcn_readlane(own.n, l),
                     __builtin_amdgcn_readlane(own.kv, l), __builtin_amdgcn_readlane((int)own.bad, l) != 0};
    }
};

// Equal contiguous ranges of `total` units over n_wgs <= total workgroups: w's
// starts at unit w * total / n_wgs, none is empty; and the one that holds unit u.
__host__ __device__ __forceinline__ int pg_start(int w, int total, int n_wgs) {
    if (n_wgs == total) return w;
    // (in 32 bits: n_wgs is at most PG_WGS here)
    const unsigned q = (unsigned)total / (unsigned)n_wgs, rest = (unsigned)total % (unsigned)n_wgs;
    return w * (int)q + (int)((unsigned)w * rest / (unsigned)n_wgs);
}
__host__ __device__ __forceinline__ int pg_owner(int u, int total, int n_wgs) {
    return (int)((((long)u + 1) * n_wgs - 1) / total);
}
__device__ __forceinline__ PgJoin pg_join(bool cut, int rows, const PgSeq& q, int head, int i0, int last_unit,
                                          int total, int n_wgs, int slot) {
    if (!cut) return PgJoin{};
    return PgJoin{rows, pg_owner(last_unit, total, n_wgs), slot, q.row0, q.kv - q.n, head, i0, 0};
}

// Calls f.run<E, T, HD>() for the types of a call.
template <class F>
hipError_t paged_with_types(int kv_dtype, int dtype, int hd, F f) {
    const bool h64 = hd == 64;
    if (kv_dtype == GGML_F16 && dtype == GGML_F32)
        return h64 ? f.template run<_Float16, float, 64>() : f.template run<_Float16, float, 128>();
    if (kv_dtype == GGML_F16 && dtype == GGML_F16)
        return h64 ? f.template run<_Float16, _Float16, 64>() : f.template run<_Float16, _Float16, 128>();
    if (kv_dtype == GGML_BF16 && dtype == GGML_F32)
        return h64 ? f.template run<__bf16, float, 64>() : f.template run<__bf16, float, 128>();
    if (kv_dtype == GGML_BF16 && dtype == GGML_BF16)
        return h64 ? f.template run<__bf16, __bf16, 64>() : f.template run<__bf16, __bf16, 128>();
    return hipErrorInvalidValue;
}

#endif  // __HIPCC__

}  // namespace frq
