// Operators of a batch of sequences over a paged KV cache (paged.hpp):
//
//   append     RoPE of the packed q and k rows (rotate-half with the f32
//              tables, as rope_append_rows), k and v rounded once to the
//              cache's type and written at each row's position
//   attention  of packed rows over the cache rows 0 .. each row's position,
//              n_heads / kv_heads query heads to a KV head
//
// Attention, one wavefront and 16 query rows of one KV head.  A sequence's
// rows and the G = n_heads / kv_heads query heads of a KV head are one list of
// n * G query rows (row i is head i % G of packed row i / G), so that grouped
// heads fill the MFMA's columns and share the K and V loads.  For 32 keys at a
// time:
//   S^T (keys x rows) = K . Q^T on v_mfma_f32_16x16x32, two groups of 16 keys.
//     The C layout leaves lane 16 g + r keys 4g + i (i < 4) of each group for
//     row r: with both groups its 8 values of the PV product's k index, in an
//     order that V's loads follow.  P never moves between lanes.
//   p = e^(s - m) and their sum l per row (l per lane until the end); m is the
//     running maximum, of f16 parts a bound of the block's own (PG_DROP)
//   O^T (dims x rows) += V^T . P^T: tile t takes the dims VW * r + t, so that
//     lane 16 g + r's loads of its 8 keys, VW dims from VW * r, hold the A
//     operand of all VW tiles, put together by byte permutes.
// f32 activations: q and p are split into parts of the cache's type (2 of f16,
// 3 of bf16), which keeps products and sums at f32's precision.  f16 parts
// take q scaled by a power of two per row (exact), its largest to 2^14 .. 2^15:
// no part leaves f16's range, and a small dim keeps steps of 2^-39 of the largest.
// 16-bit activations: q as it is, p in two parts; their products cost nothing
// here, where K and V bytes are the bound, and one part would add a rounding as
// large as the output's own.
// p carries a factor 2^TOP, which l carries too: f16 parts of small p keep steps
// of 2^-24 / 2^15 of the largest p of 32 keys.
#include <hip/hip_runtime.h>

#include "common.hpp"
#include "kernels.hpp"
#include "paged.hpp"
#include "paged_rows.hpp"

namespace frq {

namespace {

template <class E, class T, int HD>
struct Rows16 {
    using Cache = PagedKv;
    using Row = T;
    using P = PgElem<E>;
    using v8 = typename P::v8;
    static constexpr bool WIDE = std::is_same<T, float>::value;
    static constexpr int NQ = WIDE ? P::SPLIT : 1;
    static constexpr int NP = WIDE ? P::SPLIT : 2;
    static constexpr int DIM = HD, KS = HD / 32, VW = HD / 16;
    static constexpr int STEP = 32, BYTES = 2 * HD;  // keys of a block; bytes of a key
    static constexpr int RESIDENT = pg_resident(HD, 2);

    v8 q[NQ][KS];
    float factor;  // score = S^T * factor, in units of log2
    int limit;     // the row's position; -1: it sees nothing
    pg_f4 o[VW];
    float m, l, peak;  // peak: the largest score so far

    struct KeyRegs {
        pg_u4 w[2][KS];
    };
    typedef uint32_t ValueWord __attribute__((ext_vector_type(VW / 2)));
    struct ValueRegs {
        ValueWord w[8];
    };

    // Lane 16 g + r takes row r: dims 32 t + 8 g + e of x.
    __device__ void load_q(const T* x, float scale) {
        const int g = (threadIdx.x & 63) >> 4;
        pd_load_q<E>(q, factor, x, scale, [&](int t) { return 32 * t + 8 * g; });
    }

    __device__ void start() {
#pragma unroll
        for (int t = 0; t < VW; t++) o[t] = pg_f4{0.f, 0.f, 0.f, 0.f};
        m = peak = PG_LEAST;
        l = 0.0f;
    }

    // The loads of 32 keys: group a's 16 rows start at ka[a] / va[a].  ONCE:
    // nothing else of the call reads them, so they go past the caches.
    template <bool ONCE, class W>
    __device__ static W load(const E* p) {
        return ONCE ? __builtin_nontemporal_load(reinterpret_cast<const W*>(p)) : *reinterpret_cast<const W*>(p);
    }
    template <bool ONCE>
    __device__ static void load_k(KeyRegs& k, const E* const (&ka)[2]) {
        const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
#pragma unroll
        for (int a = 0; a < 2; a++)
#pragma unroll
            for (int t = 0; t < KS; t++) k.w[a][t] = load<ONCE, pg_u4>(ka[a] + r * HD + 32 * t + 8 * g);
    }
    template <bool ONCE>
    __device__ static void load_v(ValueRegs& v, const E* const (&va)[2]) {
        const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
#pragma unroll
        for (int a = 0; a < 2; a++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                v.w[4 * a + i] = load<ONCE, ValueWord>(va[a] + (4 * g + i) * HD + VW * r);
    }

    // Which keys of a block of 32 from j0 a row sees: none past its position,
    // past the sequence's length kv or in a page that is none (bad: NaN).
    struct Mask {
        int j0, kv;
        bool bad[2];
    };

    // The block's scores in log2 units: s[4 a + i] of key 16 a + 4 g + i.
    template <bool MASK>
    __device__ void scores(const KeyRegs& k, const Mask& mk, float (&s)[8]) const {
        const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
        for (int a = 0; a < 2; a++) {
            pg_f4 st = pg_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int t = 0; t < KS; t++)
#pragma unroll
                for (int p = NQ - 1; p >= 0; p--) st = P::mfma16(__builtin_bit_cast(v8, k.w[a][t]), q[p][t], st);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float v = st[i] * factor;
                if constexpr (MASK) {
                    if (mk.bad[a]) v = pg_nan();
                    if (mk.j0 + 16 * a + 4 * g + i > limit) v = -__builtin_inff();
                }
                s[4 * a + i] = v;
            }
        }
    }

    // Weights of the block's scores (s becomes them), maximum and sums renewed.
    __device__ void weights(float (&s)[8], v8 (&pp)[NP]) {
        float top = s[0];
#pragma unroll
        for (int i = 1; i < 8; i++) top = fmaxf(top, s[i]);
        top = pg_row_max(top);
        peak = fmaxf(peak, top);
        // (whole steps: c is exact)
        const float mn = std::is_same<E, _Float16>::value ? __builtin_ceilf(fmaxf(top, peak - PG_DROP)) : peak;
        const float c = __builtin_amdgcn_exp2f(m - mn);  // (0 or 1 where nothing was seen before: l = o = 0)
        m = mn;
        l *= c;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            s[i] = __builtin_amdgcn_exp2f(s[i] - mn + P::TOP);
            l += s[i];
            float rest = s[i];
#pragma unroll
            for (int p = 0; p < NP; p++) {
                pp[p][i] = (E)rest;
                rest -= (float)pp[p][i];
            }
        }
#pragma unroll
        for (int t = 0; t < VW; t++) o[t] *= c;
    }

    __device__ void product(const ValueRegs& v, const v8 (&pp)[NP]) {
#pragma unroll
        for (int t = 0; t < VW; t++) {
            const uint32_t sel = (t & 1) ? 0x07060302u : 0x05040100u;  // high or low halves of two words
            uint4 a;
            a.x = __builtin_amdgcn_perm(v.w[1][t >> 1], v.w[0][t >> 1], sel);
            a.y = __builtin_amdgcn_perm(v.w[3][t >> 1], v.w[2][t >> 1], sel);
            a.z = __builtin_amdgcn_perm(v.w[5][t >> 1], v.w[4][t >> 1], sel);
            a.w = __builtin_amdgcn_perm(v.w[7][t >> 1], v.w[6][t >> 1], sel);
#pragma unroll
            for (int p = NP - 1; p >= 0; p--) o[t] = P::mfma16(__builtin_bit_cast(v8, a), pp[p], o[t]);
        }
    }

    // Keys that no row of the sequence may see: their rows hold anything.
    __device__ static void clear(ValueRegs& v, const Mask& mk) {
        const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const bool none = mk.bad[i >> 2] || mk.j0 + 16 * (i >> 2) + 4 * g + (i & 3) >= mk.kv;
#pragma unroll
            for (int w = 0; w < VW / 2; w++)
                if (none) v.w[i][w] = 0;
        }
    }

    // Whether the block holds an infinite or NaN value, in any lane.
    __device__ static bool odd(const KeyRegs& k, const ValueRegs& v) {
        bool any = false;
#pragma unroll
        for (int a = 0; a < 2; a++)
#pragma unroll
            for (int t = 0; t < KS; t++)
#pragma unroll
                for (int w = 0; w < 4; w++) any |= pg_word_odd<E>(k.w[a][t][w]);
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
            for (int w = 0; w < VW / 2; w++) any |= pg_word_odd<E>(v.w[i][w]);
        return __any(any);
    }

    // Keys [j0, j1) by pg_plain(); x: the row's q.
    __device__ void plain(const PagedKv& c, const int* table, int head, const T* x, float scale, int j0, int j1) {
        const int g = (threadIdx.x & 63) >> 4;
        pg_plain<PgCells<E, HD>, T, HD, 4>(
            c, table, head, x, scale, limit, j0, j1, [](float x) { return x; }, P::TOP, g == 0,
            [&](int i) { return 4 * (VW * g + i); },
            [&](int i, int e, float f, float p, float v) {
                const int t = (4 * i + e) % VW, k = (4 * i + e) / VW;
                o[t][k] = fmaf(p, v, o[t][k] * f);
            },
            m, l);
        peak = fmaxf(peak, m);
    }

    // One wavefront over keys [j0, j1) of a sequence of kv (j0 a multiple of 32).
    // The next block's keys are loaded as soon as this one's scores are formed, its
    // values as soon as this one's product is: one or the other is in flight all
    // the time, in one set of registers each (two sets spill at HD 128).  The page
    // ids of 1024 keys are one load, lane i holding the page of group i.  Every row
    // sees the keys up to all_see.
    template <bool ONCE>
    __device__ __forceinline__ void walk(const PagedKv& c, const int* table, int head, int j0, int j1, int kv, int all_see) {
        const int lane = threadIdx.x & 63;
        while (j0 < j1) {
            const int end = min(j1, j0 + 1024);
            const int jl = j0 + 16 * lane;
            bool off;
            const int page = pg_page(c, table, jl, kv, off);
            const uint64_t none = __ballot(off && jl < end);  // groups whose page is none
            auto rows = [&](const void* pool, int blk, const E* (&at)[2]) {
    #pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int g = 2 * blk + i, p = __builtin_amdgcn_readlane(page, g);
                    at[i] = static_cast<const E*>(pool) + ((((size_t)p * c.kv_heads + head) << c.log_ps) +
                                                           ((j0 + 16 * g) & ((1 << c.log_ps) - 1))) * HD;
                }
            };
            const int last = (end - j0 + 31) / 32 - 1;
            const E* at[2];
            KeyRegs kr;
            ValueRegs vr;
            float s[8];
            v8 pp[NP];
            rows(c.k, 0, at);
            load_k<ONCE>(kr, at);
            rows(c.v, 0, at);
            load_v<ONCE>(vr, at);
            for (int i = 0;; i++) {
                const int j = j0 + 32 * i;
                const uint32_t bad = (uint32_t)(none >> (2 * i)) & 3;
                const Mask mk{j, kv, {(bad & 1) != 0, (bad & 2) != 0}};
                const bool mask = j + 31 > all_see || bad;
                if (i == last || mask) {  // (apart from the loop's body, which keeps its loads in flight)
                    if (mask) scores<true>(kr, mk, s);
                    else scores<false>(kr, mk, s);
                    weights(s, pp);
                    if (mask) clear(vr, mk);
                    product(vr, pp);
                    if (i == last) break;
                    rows(c.k, i + 1, at);
                    load_k<ONCE>(kr, at);
                    rows(c.v, i + 1, at);
                    load_v<ONCE>(vr, at);
                    continue;
                }
                scores<false>(kr, mk, s);
                rows(c.k, i + 1, at);
                load_k<ONCE>(kr, at);
                weights(s, pp);
                product(vr, pp);
                rows(c.v, i + 1, at);
                load_v<ONCE>(vr, at);
            }
            j0 = end;
        }
    }

    // The same keys once more, if their sums hold an infinite or NaN value: blocks of
    // such values or of pages that are none one key after another.  64 sequences of up to
    // 8191, a call waited for: 85 us, with one infinite value 120, with one in every 16
    // keys 550, all NaN 225.
    __device__ __forceinline__ void walk_odd(const PagedKv& c, const int* table, int head, int j0, int j1, int kv, const T* x,
                                             float scale) {
        if (!__any(pg_odd(o))) return;
        start();
    #pragma unroll 1
        for (int j = j0; j < j1; j += 32) {
            Mask mk{j, kv, {}};
            const E *ka[2], *va[2];
    #pragma unroll
            for (int i = 0; i < 2; i++) {
                const size_t page = pg_page(c, table, j + 16 * i, kv, mk.bad[i]);
                const size_t at = (((page * c.kv_heads + head) << c.log_ps) + ((j + 16 * i) & ((1 << c.log_ps) - 1))) * HD;
                ka[i] = static_cast<const E*>(c.k) + at;
                va[i] = static_cast<const E*>(c.v) + at;
            }
            KeyRegs kr;
            ValueRegs vr;
            load_k<false>(kr, ka);
            load_v<false>(vr, va);
            clear(vr, mk);
            if (mk.bad[0] || mk.bad[1] || odd(kr, vr)) {
                plain(c, table, head, x, scale, j, min(j + 32, j1));
                if (__all(pg_all_nan(o))) return;
                continue;
            }
            float s[8];
            v8 pp[NP];
            scores<true>(kr, mk, s);
            weights(s, pp);
            product(vr, pp);
        }
    }

    // The row's sum over the four lanes that share it.
    __device__ void finish() {
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
    }
};

// Joins the pieces of cut tiles: workgroups (x, y) take rows wg_rows y .. of the
// one that workgroup x left to be joined, if it left one, or with fewer x than
// records of the x-th that is left at all.  HD / 4 threads a row, as many groups
// of such threads as there is room for with every so many-th piece each, PJ_STEP
// pieces a step, whose loads are one memory round trip.
constexpr int PJ_WG = 256;
template <class T, int HD, int PJ_STEP, bool NORMALIZED>
__global__ __launch_bounds__(PJ_WG) void paged_join_kernel(const PgJoin* __restrict__ joins, int records,
                                                           const float* __restrict__ part, int tile_rows, int wg_rows,
                                                           int grp, T* __restrict__ out, int ldo) {
    constexpr int TH = HD / 4;
    __shared__ pg_f4 s_o[PJ_WG];
    __shared__ float s_l[PJ_WG / TH], s_m[PJ_WG / TH];
    __shared__ uint64_t s_some[PG_RECORDS / 64];
    int w0 = blockIdx.x;
    if ((int)gridDim.x < records) {
        for (int i = threadIdx.x; i < PG_RECORDS; i += PJ_WG) {
            const uint64_t some = __ballot(i < records && joins[i].rows > 0);
            if ((threadIdx.x & 63) == 0) s_some[i >> 6] = some;
        }
        __syncthreads();
        int skip = blockIdx.x, k = 0;
        for (; k < PG_RECORDS / 64 && skip >= __popcll(s_some[k]); k++) skip -= __popcll(s_some[k]);
        if (k == PG_RECORDS / 64) return;
        uint64_t some = s_some[k];
        for (; skip; skip--) some &= some - 1;
        w0 = __builtin_amdgcn_readfirstlane(64 * k + __builtin_ctzll(some));
    }
    const PgJoin j = joins[w0];
    const int r0 = wg_rows * blockIdx.y, rows = min(wg_rows, j.rows - r0);
    if (rows <= 0) return;
    const int groups = (unsigned)(PJ_WG / TH) / (unsigned)rows;
    const int d = threadIdx.x % TH, x = threadIdx.x / TH, p = (unsigned)x / (unsigned)rows, r = r0 + x - p * rows;
    const float* row = part + r * HD + 4 * d;
    const float* stat = part + tile_rows * HD + r;
    float M = PG_LEAST, L = 0.0f;
    pg_f4 O = pg_f4{0.f, 0.f, 0.f, 0.f};
    if (p < groups) {
        for (int w = w0 + p; w <= j.last; w += groups * PJ_STEP) {
            pg_f4 o[PJ_STEP];
            float m[PJ_STEP], l[PJ_STEP], mn = M;
#pragma unroll
            for (int i = 0; i < PJ_STEP; i++) {  // (past the last: the last again, not added)
                const int wi = min(w + i * groups, j.last);
                const size_t slot = (size_t)(wi == w0 ? j.slot : 2 * wi) * pg_slot(tile_rows, HD);
                o[i] = *reinterpret_cast<const pg_f4*>(row + slot);
                m[i] = stat[slot];
                l[i] = stat[slot + tile_rows];
            }
#pragma unroll
            for (int i = 0; i < PJ_STEP; i++) mn = fmaxf(mn, m[i]);
            const float f = __builtin_amdgcn_exp2f(M - mn), was = L;
            M = mn;
            L *= f;
            float e[PJ_STEP];
#pragma unroll
            for (int i = 0; i < PJ_STEP; i++) {
                e[i] = __builtin_amdgcn_exp2f(m[i] - mn);
                L = fmaf(l[i], w + i * groups <= j.last ? e[i] : 0.0f, L);
            }
            O *= pg_factor<NORMALIZED>(f, was, L);
#pragma unroll
            for (int i = 0; i < PJ_STEP; i++) {
                const bool add = w + i * groups <= j.last;
                const float x = pg_factor<NORMALIZED>(e[i], l[i], L);
#pragma unroll
                for (int k = 0; k < 4; k++) O[k] = add ? fmaf(o[i][k], x, O[k]) : O[k];  // (o may be infinite)
            }
        }
        s_o[threadIdx.x] = O;
        if (d == 0) {
            s_l[x] = L;
            s_m[x] = M;
        }
    }
    __syncthreads();
    if (p) return;
    float mx = PG_LEAST;
    for (int i = 0; i < groups; i++) mx = fmaxf(mx, s_m[i * rows + x]);
    L = 0.0f;
    O = pg_f4{0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < groups; i++) L = fmaf(s_l[i * rows + x], __builtin_amdgcn_exp2f(s_m[i * rows + x] - mx), L);
    for (int i = 0; i < groups; i++) {
        const float e = pg_factor<NORMALIZED>(__builtin_amdgcn_exp2f(s_m[i * rows + x] - mx), s_l[i * rows + x], L);
        const pg_f4 o = s_o[(i * rows + x) * TH + d];
#pragma unroll
        for (int k = 0; k < 4; k++) O[k] = fmaf(o[k], e, O[k]);
    }
    L = pg_divisor<NORMALIZED>(L);
    const int at = (unsigned)(j.i0 + r) / (unsigned)grp;
    const size_t to = j.row0 + at, h = j.head * grp + (j.i0 + r - at * grp);
    T y[4];
#pragma unroll
    for (int k = 0; k < 4; k++) y[k] = (T)(j.pos0 + at < 0 ? 0.0f : O[k] / L);
    __builtin_memcpy(__builtin_assume_aligned(out + to * ldo + h * HD + 4 * d, 8), y, sizeof y);
}

// Append.  Workgroups (row, y): the row's work in chunks, AP_WG of them a
// workgroup and turn: 8 pairs (elements i .. i + 7 and i + HD / 2 ..) of a head
// of q or k, or 8 elements of v, each 16 or 32 bytes a lane.
//   y[i] = x[i] cos[i] - x[i + HD/2] sin[i],
//   y[i + HD/2] = x[i + HD/2] cos[i + HD/2] + x[i] sin[i + HD/2]
// (rope_f32, byte_kernels.rs:1885-1964): two products and a sum in f32, rounded
// once.  A thread's chunks are the same part of different heads, so it reads
// its part of the position's table rows once.  A chunk's loads need the row
// alone and go out before the row's sequence and position are known.
// Bound by HBM for many rows (12254 of f32, 32 heads over 8 of 128: 554 MB in
// 102 us), by three memory round trips for few (row_start and kv_len, page and table
// rows, the stores; 2.8 us for one, 4.0 for 256).
constexpr int AP_WG = 256;
constexpr int AP_FEW = 2048;
template <class E, class T, int HD>
__global__ __launch_bounds__(AP_WG) void paged_append_kernel(PagedKv c, PagedRows b, int n_heads,
                                                             const T* q, int ldq, const T* __restrict__ k, int ldk,
                                                             const T* __restrict__ v, int ldv,
                                                             const float* __restrict__ cs, const float* __restrict__ sn,
                                                             int rope_rows, T* q_out, int ldqo) {
    constexpr int HALF = HD / 2, CP = HALF / 8;  // chunks of a head
    const int row = blockIdx.x, nq = q ? n_heads : 0;
    const int turned = CP * (nq + c.kv_heads), all = turned + 2 * CP * c.kv_heads;
    const int stride = AP_WG * gridDim.y;  // (a multiple of CP)
    int e = AP_WG * blockIdx.y + threadIdx.x;
    const int i = 8 * (e % CP);
    T lo[8], hi[8];
    auto fetch = [&] {
        if (e < turned) {
            const int h = e / CP;
            const T* x = h < nq ? q + (size_t)row * ldq + h * HD : k + (size_t)row * ldk + (h - nq) * HD;
            __builtin_memcpy(lo, __builtin_assume_aligned(x + i, 16), sizeof lo);
            __builtin_memcpy(hi, __builtin_assume_aligned(x + i + HALF, 16), sizeof hi);
        } else if (e < all) {
            __builtin_memcpy(lo, __builtin_assume_aligned(v + (size_t)row * ldv + 8 * (e - turned), 16), sizeof lo);
        }
    };
    fetch();
    const int s = pg_row_seq(b, row);
    if (s < 0) return;
    const PgSeq sq = pg_seq(b, s);
    if (row < sq.row0 || row >= sq.row0 + sq.n) return;
    const int pos = sq.kv - sq.n + (row - sq.row0);
    const bool bad = sq.bad || (cs && pos >= rope_rows), seen = pos >= 0 && !bad;
    const int page = seen ? b.table[(size_t)s * b.max_pages + (pos >> c.log_ps)] : -1;
    float cl[8], ch[8], sl[8], sh[8];
    if (cs && seen && e < turned) {
        const float *ct = cs + (size_t)pos * HD + i, *st = sn + (size_t)pos * HD + i;
        __builtin_memcpy(cl, __builtin_assume_aligned(ct, 16), sizeof cl);
        __builtin_memcpy(ch, __builtin_assume_aligned(ct + HALF, 16), sizeof ch);
        __builtin_memcpy(sl, __builtin_assume_aligned(st, 16), sizeof sl);
        __builtin_memcpy(sh, __builtin_assume_aligned(st + HALF, 16), sizeof sh);
    }
    const bool put = (unsigned)page < (unsigned)c.n_pages;
    const size_t at = (((size_t)(put ? page : 0) * c.kv_heads) << c.log_ps) + (pos & ((1 << c.log_ps) - 1));
    auto cache_row = [&](void* pool, int h) { return static_cast<E*>(pool) + (at + ((size_t)h << c.log_ps)) * HD; };
    for (; e < all; e += stride, fetch()) {
        if (e >= turned) {
            if (!put) continue;
            const int x = 8 * (e - turned);
            E y[8];
#pragma unroll
            for (int j = 0; j < 8; j++) y[j] = (E)(float)lo[j];
            __builtin_memcpy(__builtin_assume_aligned(cache_row(c.v, x / HD) + x % HD, 16), y, sizeof y);
            continue;
        }
        const int h = e / CP;
        float a[8], z[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            a[j] = (float)lo[j];
            z[j] = (float)hi[j];
        }
        if (cs && seen) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float x = a[j], y = z[j];
                a[j] = x * cl[j] - y * sl[j];
                z[j] = y * ch[j] + x * sh[j];
            }
        }
        if (h < nq) {
            T y[8], x[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                y[j] = (T)(bad ? pg_nan() : pos < 0 ? 0.0f : a[j]);
                x[j] = (T)(bad ? pg_nan() : pos < 0 ? 0.0f : z[j]);
            }
            T* to = q_out + (size_t)row * ldqo + h * HD + i;
            __builtin_memcpy(__builtin_assume_aligned(to, 16), y, sizeof y);
            __builtin_memcpy(__builtin_assume_aligned(to + HALF, 16), x, sizeof x);
        } else if (put) {
            E y[8], x[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                y[j] = (E)a[j];
                x[j] = (E)z[j];
            }
            E* to = cache_row(c.k, h - nq) + i;
            __builtin_memcpy(__builtin_assume_aligned(to, 16), y, sizeof y);
            __builtin_memcpy(__builtin_assume_aligned(to + HALF, 16), x, sizeof x);
        }
    }
}

struct AppendCall {
    const PagedAppendArgs& p;
    hipStream_t s;
    template <class E, class T, int HD>
    hipError_t run() const {
        // one chunk a thread while that does not fill the chip
        const int chunks = HD / 16 * ((p.q ? p.n_heads : 0) + 3 * p.kv.kv_heads), parts = (chunks + AP_WG - 1) / AP_WG;
        const int y = (long)p.rows.rows * parts <= AP_FEW ? parts : 1;
        hipLaunchKernelGGL((paged_append_kernel<E, T, HD>), dim3(p.rows.rows, y), dim3(AP_WG), 0, s, p.kv, p.rows,
                           p.n_heads, static_cast<const T*>(p.q), p.ldq, static_cast<const T*>(p.k), p.ldk,
                           static_cast<const T*>(p.v), p.ldv, p.cos, p.sin, p.rope_rows, static_cast<T*>(p.q_out),
                           p.ldqo);
        return hipGetLastError();
    }
};

// wgs: workgroups that may have left pieces, of at most `tiles` tiles with
// `rows` rows.  Tiles of 128 rows, few (in four pieces or more each): 8 pieces a
// step, and only as many workgroups as there are tiles, since empty ones of more
// than the chip holds at a time take their turn as well: 16 tiles in 32 pieces
// 54.5 -> 8.3 us, 64 in 8 22.4 -> 10.7 (of 256 in 2 or 3, where most workgroups
// have one, finding it costs more: 18.2 -> 23.5).  Tiles of 16 rows in many pieces
// each, a row a workgroup: 2 sequences of 29561, 128 pieces, 28.9 -> 22.7 us a whole
// call; one of 131071, 8 KV heads, 64 pieces, 92.6 -> 91.2.
template <class T, int HD, bool NORMALIZED>
hipError_t join(const PgJoin* joins, const float* part, int wgs, long tiles, int tile_rows, int rows, int grp,
                void* out, int ldo, hipStream_t s) {
    const bool few = tiles <= wgs / 4;
    const auto kernel = tile_rows == 16 || few ? paged_join_kernel<T, HD, 8, NORMALIZED>
                                                : paged_join_kernel<T, HD, 2, NORMALIZED>;
    const int wg_rows = tile_rows == 16 && tiles <= wgs / 32 ? 1 : 4, y = (rows + wg_rows - 1) / wg_rows;
    const int x = few && wgs * y > 2048 ? (int)tiles : wgs;
    hipLaunchKernelGGL(kernel, dim3(x, y), dim3(PJ_WG), 0, s, joins, wgs, part, tile_rows, wg_rows, grp,
                       static_cast<T*>(out), ldo);
    return hipGetLastError();
}

struct Rows16Call {
    const PagedAttendArgs& p;
    hipStream_t s;
    template <class E, class T, int HD>
    hipError_t run() const {
        return rows16_launch<Rows16<E, T, HD>>(p, p.kv, s);
    }
};

}  // namespace

size_t paged_rows16_work_bytes(const PagedKv& kv, const PagedRows& r, int n_heads, int hd) {
    return rows16_work_bytes(kv, r, n_heads, hd, 2);
}

bool paged_rows16_fits(const PagedKv& kv, const PagedRows& r, int n_heads, int hd) {
    return rows16_fits(kv, r, n_heads, hd, 2);
}

bool paged_types(int kv_dtype, int dtype) {
    return (kv_dtype == GGML_F16 && (dtype == GGML_F32 || dtype == GGML_F16)) ||
           (kv_dtype == GGML_BF16 && (dtype == GGML_F32 || dtype == GGML_BF16));
}

hipError_t launch_paged_append(int kv_dtype, int dtype, int hd, const PagedAppendArgs& p, hipStream_t s) {
    if (p.rows.rows <= 0) return hipSuccess;
    return paged_with_types(kv_dtype, dtype, hd, AppendCall{p, s});
}

hipError_t launch_paged_join(int dtype, int hd, const PgJoin* joins, const float* part, int wgs, long tiles,
                             int tile_rows, int rows, int grp, bool normalized, void* out, int ldo, hipStream_t s) {
    const auto run =
        dtype == GGML_F32 && normalized   ? (hd == 64 ? join<float, 64, true> : join<float, 128, true>)
        : dtype == GGML_F32               ? (hd == 64 ? join<float, 64, false> : join<float, 128, false>)
        : dtype == GGML_F16 && normalized ? (hd == 64 ? join<_Float16, 64, true> : join<_Float16, 128, true>)
        : dtype == GGML_F16               ? (hd == 64 ? join<_Float16, 64, false> : join<_Float16, 128, false>)
                                          : (hd == 64 ? join<__bf16, 64, false> : join<__bf16, 128, false>);
    return run(joins, part, wgs, tiles, tile_rows, rows, grp, out, ldo, s);
}

hipError_t launch_paged_rows16(int kv_dtype, int dtype, int hd, const PagedAttendArgs& p, hipStream_t s) {
    if (p.rows.rows <= 0 || p.rows.n_seqs <= 0) return hipSuccess;
    return paged_with_types(kv_dtype, dtype, hd, Rows16Call{p, s});
}

}  // namespace frq
