// Operators of a batch of sequences over an 8-bit paged KV cache (paged8.hpp):
// append, and attention of few rows a sequence.
//
// Append.  e4m3 has a relative step of 2^-4 .. 2^-3 between its least normal number
// and its largest, so a block of 16 positions of a head needs a power of two alone:
//   2^e, the least for which its largest |value| is at most 448 * 2^e
// (e from -127 to 120).  Rows that join older ones in their block take the block's
// scale, or raise it: then the older codes are rounded once more, exactly but for
// those that fall below the least normal number, 2^-6 in units of the new scale: 2^-13.8
// of the block's largest, which is above 224 of them.
//
// Attention: as paged.hip's 16-row tiles, 32 keys at a time.  K's codes go to the
// matrix pipe as f16 (bf16 for bf16 rows) without their scale, exactly; a group of
// 16 keys' scale is a factor of its scores, in f32.  V's go there as bf16 values,
// exactly, so that no weight has to carry a scale.  f32 rows: q in two parts of f16,
// 16-bit rows as they are; weights in two parts of bf16, to 2^-16 of each (V's codes
// are 2^-4 of what was appended), for f32 rows in three, to f32's own precision: the
// third costs 1 % (96 sequences of up to 7942, f32, 82 us).
// Bound by HBM and some 10 us beside it: the lookup and the first keys, the join.  32
// heads over 8 of 128: one sequence of 200002, 410 MB, 75 us (70 with the loads
// alone); 96 of up to 7942, 333 MB, 82 (68 alone); 64 heads over 8 of 64, 128 of 307 ..
// 2489, 132 MB, 36 (32 alone).  One of 901, 32 KV heads: 10 us, 7 of them the two
// launches' start.
// No faster: blocks of 64 keys, three workgroups a CU for dims of 128, the odd blocks'
// code out of line.
#include <hip/hip_runtime.h>

#include "common.hpp"
#include "kernels.hpp"
#include "paged8.hpp"
#include "paged_rows.hpp"

namespace frq {

namespace {

template <class T, int HD>
struct Rows8 {
    using Cache = PagedKv8;
    using Row = T;
    static constexpr bool WIDE = std::is_same<T, float>::value;
    using E = typename std::conditional<WIDE, _Float16, T>::type;  // of q and k in their products
    using P = PgElem<__bf16>;                                      // of weights and v
    using q8 = typename PgElem<E>::v8;
    using v8 = P::v8;
    static constexpr int NQ = WIDE ? 2 : 1, NP = WIDE ? 3 : 2;
    static constexpr int DIM = HD, KS = HD / 32, VW = HD / 16;
    // Groups of 16 keys of a block.  (Of four, where the 16 KB of two blocks of 32 go
    // out at once: no faster, and 10.0 us for 7.6 where a wavefront has a few blocks.)
    static constexpr int G = 2, STEP = 16 * G, BYTES = HD;
    // Workgroups a CU.  Dims of 64: 512 workgroups of them 38.7 us, 768 31.8, 1024 35.7
    // (128 sequences of 308 .. 2489, 8 KV heads); of 128: 83.8, 93.3, 131 (spills).
    static constexpr int RESIDENT = pg_resident(HD, 1);
    // Weights are 2^TOP at most; the maximum that they are of is renewed where scores
    // pass it by LAZY: bf16 weights keep their digits whatever power of two they and
    // the sums share.
    static constexpr float LAZY = 7.0f, SHIFT = P::TOP - LAZY;

    q8 q[NQ][KS];
    float factor;  // score = product * factor * the key's scale, in units of log2
    int limit;     // the row's position; -1: it sees nothing
    pg_f4 o[VW];
    float m, l;

    typedef uint32_t ValueWord __attribute__((ext_vector_type(VW / 4)));
    struct KeyRegs {
        pg_u4 w[G][HD / 64];
    };
    struct ValueRegs {
        ValueWord w[4 * G];
    };

    // Lane 16 g + r takes row r: in step t of the products dims 64 (t / 2) + 16 g +
    // 8 (t % 2) + e, so that a lane's 16 codes of a key are one load.
    __device__ void load_q(const T* x, float scale) {
        const int g = (threadIdx.x & 63) >> 4;
        pd_load_q<E>(q, factor, x, scale, [&](int t) { return 64 * (t >> 1) + 16 * g + 8 * (t & 1); });
    }

    __device__ void start() {
#pragma unroll
        for (int t = 0; t < VW; t++) o[t] = pg_f4{0.f, 0.f, 0.f, 0.f};
        m = PG_LEAST;
        l = 0.0f;
    }

    // The loads of a block of keys: group a's 16 rows start at at[a], values' loads
    // are those of groups 2 h and 2 h + 1.  ONCE: nothing else of the call reads them,
    // so they go past the caches.
    using Base = const P8Global<uint8_t>*;
    template <bool ONCE, class W>
    __device__ static W load(Base p) {
        const auto* w = reinterpret_cast<const P8Global<W>*>(p);
        return ONCE ? __builtin_nontemporal_load(w) : *w;
    }
    template <bool ONCE>
    __device__ static void load_k(KeyRegs& k, const Base (&at)[G]) {
        const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
#pragma unroll
        for (int a = 0; a < G; a++)
#pragma unroll
            for (int c = 0; c < HD / 64; c++) k.w[a][c] = load<ONCE, pg_u4>(at[a] + r * HD + 64 * c + 16 * g);
    }
    template <bool ONCE>
    __device__ static void load_v(ValueRegs& v, const Base (&at)[G], int h) {
        const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
#pragma unroll
        for (int a = 2 * h; a < 2 * h + 2; a++)
#pragma unroll
            for (int i = 0; i < 4; i++) v.w[4 * a + i] = load<ONCE, ValueWord>(at[a] + (4 * g + i) * HD + VW * r);
    }

    // What holds for the groups of a block from key j0: their scales (2^0 for groups
    // without keys, so that what is cleared stays 0), and which keys a row sees: none
    // past its position, past the sequence's length kv or in a page that is none (bad:
    // NaN).
    struct Block {
        int j0, kv, ks[G], vs[G];
        uint32_t bad;
    };

    // The block's scores in log2 units: s[4 a + i] of key 16 a + 4 g + i.
    __device__ void scores(const KeyRegs& k, const Block& b, float (&s)[4 * G]) const {
#pragma unroll
        for (int a = 0; a < G; a++) {
            pg_f4 st = pg_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int t = 0; t < KS; t++) {
                const q8 x = p8_eight<E>(k.w[a][t >> 1][2 * (t & 1)], k.w[a][t >> 1][2 * (t & 1) + 1], 1.0f);
#pragma unroll
                for (int p = NQ - 1; p >= 0; p--) st = PgElem<E>::mfma16(x, q[p][t], st);
            }
            const float unit = p8_factor(b.ks[a]);
#pragma unroll
            for (int i = 0; i < 4; i++) s[4 * a + i] = st[i] * factor * unit;
            if (a & 1) __builtin_amdgcn_sched_barrier(0);  // (all of a block's at once spill)
        }
    }
    // Those of keys that the row does not see.
    __device__ void hide(const Block& b, float (&s)[4 * G]) const {
        const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
        for (int i = 0; i < 4 * G; i++) {
            if ((b.bad >> (i >> 2)) & 1) s[i] = pg_nan();
            if (b.j0 + 16 * (i >> 2) + 4 * g + (i & 3) > limit) s[i] = -__builtin_inff();
        }
    }

    __device__ void renew(const float (&s)[4 * G]) {
        float top = s[0];
#pragma unroll
        for (int i = 1; i < 4 * G; i++) top = fmaxf(top, s[i]);
        top = pg_row_max(top);
        if (!__any(top > m + LAZY)) return;
        const float mn = fmaxf(m, top);
        const float c = __builtin_amdgcn_exp2f(m - mn);  // (0 or 1 where nothing was seen before: l = o = 0)
        m = mn;
        l *= c;
#pragma unroll
        for (int t = 0; t < VW; t++) o[t] *= c;
    }

    // Weights of groups 2 h and 2 h + 1 and their product with V.
    __device__ void product(const float (&s)[4 * G], const ValueRegs& v, const Block& b, int h) {
        v8 pp[NP];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            float rest = __builtin_amdgcn_exp2f(s[8 * h + i] - m + SHIFT);
            l += rest;
#pragma unroll
            for (int p = 0; p < NP; p++) {
                pp[p][i] = (__bf16)rest;
                rest -= (float)pp[p][i];
            }
        }
#pragma unroll
        for (int w = 0; w < VW / 4; w++) {
            uint32_t x[8][2];  // pairs of dims of 8 keys
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float operand = p8_operand(b.vs[2 * h + (i >> 2)]);
                x[i][0] = p8_pair<false>(v.w[8 * h + i][w], operand, __bf16());
                x[i][1] = p8_pair<true>(v.w[8 * h + i][w], operand, __bf16());
            }
#pragma unroll
            for (int t = 0; t < 4; t++) {
                const uint32_t sel = (t & 1) ? 0x07060302u : 0x05040100u;  // high or low halves of two words
                pg_u4 a;
#pragma unroll
                for (int i = 0; i < 4; i++) a[i] = __builtin_amdgcn_perm(x[2 * i + 1][t >> 1], x[2 * i][t >> 1], sel);
#pragma unroll
                for (int p = NP - 1; p >= 0; p--)
                    o[4 * w + t] = P::mfma16(__builtin_bit_cast(v8, a), pp[p], o[4 * w + t]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }

    // Keys that no row of the sequence may see: their rows hold anything.
    __device__ static void clear(ValueRegs& v, const Block& b) {
        const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
        for (int i = 0; i < 4 * G; i++) {
            const bool none = ((b.bad >> (i >> 2)) & 1) || b.j0 + 16 * (i >> 2) + 4 * g + (i & 3) >= b.kv;
#pragma unroll
            for (int w = 0; w < VW / 4; w++)
                if (none) v.w[i][w] = 0;
        }
    }

    // Whether the block holds a NaN, or values beyond f32's range, in any lane.
    __device__ static bool odd(const KeyRegs& k, const ValueRegs& v, const Block& b) {
        bool any = b.bad;
#pragma unroll
        for (int a = 0; a < G; a++) {
            any |= b.ks[a] > P8_TOP || b.vs[a] > P8_TOP;
#pragma unroll
            for (int c = 0; c < HD / 64; c++)
#pragma unroll
                for (int w = 0; w < 4; w++) any |= p8_word_nan(k.w[a][c][w]);
        }
#pragma unroll
        for (int i = 0; i < 4 * G; i++)
#pragma unroll
            for (int w = 0; w < VW / 4; w++) any |= p8_word_nan(v.w[i][w]);
        return __any(any);
    }

    // Keys [j0, j1) as pg_plain() takes them, one at a time: the registers that four
    // would take are those of a third workgroup on a CU.  x: the row's q.
    __device__ void plain(const PagedKv8& c, const int* table, int head, const T* x, float scale, int j0, int j1) {
        const int g = (threadIdx.x & 63) >> 4;
        const float unit = scale * 1.4426950408889634f;
#pragma unroll 1
        for (int j = j0; j < j1; j++) {
            bool none;
            const int page = pg_page(c, table, j, j + 1, none);
            const P8Cells<HD> cell(c, page, head, j);
            float s = 0.0f;
#pragma unroll 1
            for (int d = 4 * VW * g; d < 4 * VW * (g + 1); d += 4) {
                float y[4];
                cell.key(0, d, y);
#pragma unroll
                for (int e = 0; e < 4; e++) s = fmaf((float)x[d + e] * unit, y[e], s);
            }
            s += __shfl_xor(s, 16);
            s += __shfl_xor(s, 32);
            if (none) s = pg_nan();
            const bool sees = j <= limit;  // (no branch: the sums would be in registers twice)
            const float mn = sees ? fmaxf(m, s) : m, f = __builtin_amdgcn_exp2f(m - mn);
            const float p = __builtin_amdgcn_exp2f(s - mn + SHIFT);
            m = mn;
            l = l * f + (sees && g == 0 ? p : 0.0f);
#pragma unroll
            for (int i = 0; i < VW; i++) {
                float y[4];
                cell.value(0, 4 * (VW * g + i), y);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int t = (4 * i + e) % VW, k = (4 * i + e) / VW;
                    o[t][k] = sees ? fmaf(p, y[e], o[t][k] * f) : o[t][k];
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }

    // Block i of the groups from j0 on.
    __device__ static Block block(const P8Groups& gr, int j0, int i, int kv) {
        Block b{j0 + STEP * i, kv, {}, {}, (uint32_t)(gr.none >> (G * i)) & ((1u << G) - 1)};
#pragma unroll
        for (int a = 0; a < G; a++) {
            const bool keys = b.j0 + 16 * a < kv && !((b.bad >> a) & 1);
            b.ks[a] = keys ? __builtin_amdgcn_readlane(gr.k_scale, G * i + a) : P8_ONE;
            b.vs[a] = keys ? __builtin_amdgcn_readlane(gr.v_scale, G * i + a) : P8_ONE;
        }
        return b;
    }
    __device__ static void rows(const P8Groups& gr, const void* pool, int i, Base (&at)[G]) {
#pragma unroll
        for (int a = 0; a < G; a++) at[a] = p8_base(pool, gr.at(G * i + a));
    }

    // One wavefront over keys [j0, j1) of a sequence of kv (j0 a multiple of STEP).
    // The next block's keys are loaded as soon as this one's scores are formed, its
    // values as soon as this one's product is.  Every row sees the keys up to all_see.
    template <bool ONCE>
    __device__ __forceinline__ void walk(const PagedKv8& c, const int* table, int head, int j0, int j1, int kv,
                                         int all_see) {
        while (j0 < j1) {
            const int end = min(j1, j0 + 1024);
            P8Groups gr;
            gr.load<HD>(c, table, head, j0, kv);
            const int last = (end - j0 + STEP - 1) / STEP - 1;
            Base at[G];
            KeyRegs kr;
            ValueRegs vr;
            rows(gr, c.k, 0, at);
            load_k<ONCE>(kr, at);
            rows(gr, c.v, 0, at);
#pragma unroll
            for (int h = 0; h < G / 2; h++) load_v<ONCE>(vr, at, h);
            const auto step = [&](int i, auto more) {
                constexpr bool MORE = decltype(more)::value;
                const Block b = block(gr, j0, i, kv);
                const bool mask = b.j0 + STEP - 1 > all_see || b.bad;
                float s[4 * G];
                scores(kr, b, s);
                if constexpr (MORE) {
                    rows(gr, c.k, i + 1, at);
                    load_k<ONCE>(kr, at);
                    rows(gr, c.v, i + 1, at);
                }
                __builtin_amdgcn_sched_barrier(0);
                if (__builtin_expect(mask, 0)) hide(b, s);
                renew(s);
                if (__builtin_expect(mask, 0)) clear(vr, b);
#pragma unroll
                for (int h = 0; h < G / 2; h++) {
                    product(s, vr, b, h);
                    if constexpr (MORE) load_v<ONCE>(vr, at, h);
                    __builtin_amdgcn_sched_barrier(0);
                }
            };
            for (int i = 0; i < last; i++) step(i, std::true_type{});
            step(last, std::false_type{});
            j0 = end;
        }
    }

    // The same keys once more, if their sums hold an infinite or NaN value: blocks of
    // such values or of pages that are none one key after another.
    __device__ __forceinline__ void walk_odd(const PagedKv8& c, const int* table, int head, int j0, int j1, int kv,
                                             const T* x, float scale) {
        if (__builtin_expect(!__any(pg_odd(o)), 1)) return;
        start();
#pragma unroll 1
        for (int j = j0; j < j1; j += STEP) {
            P8Groups gr;
            gr.load<HD>(c, table, head, j, kv);
            const Block b = block(gr, j, 0, kv);
            Base ka[G], va[G];
            rows(gr, c.k, 0, ka);
            rows(gr, c.v, 0, va);
            KeyRegs kr;
            ValueRegs vr;
            load_k<false>(kr, ka);
#pragma unroll
            for (int h = 0; h < G / 2; h++) load_v<false>(vr, va, h);
            clear(vr, b);
            if (odd(kr, vr, b)) {
                plain(c, table, head, x, scale, j, min(j + STEP, j1));
                if (__all(pg_all_nan(o))) return;
                continue;
            }
            float s[4 * G];
            scores(kr, b, s);
            hide(b, s);
            renew(s);
#pragma unroll
            for (int h = 0; h < G / 2; h++) product(s, vr, b, h);
        }
    }

    // The row's sum over the four lanes that share it.
    __device__ void finish() {
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
    }
};

struct Rows8Call {
    const PagedAttendArgs& p;
    const PagedKv8& c;
    hipStream_t s;
    template <class T, int HD>
    hipError_t run() const {
        return rows16_launch<Rows8<T, HD>>(p, c, s);
    }
};

// ---- append ----

// The scale byte of values of at most amax (finite).
__device__ __forceinline__ int p8_scale_of(float amax) {
    const uint32_t u = __builtin_bit_cast(uint32_t, amax);
    // 448 = 1.75 * 2^8: exponent - 8, one more where the mantissa is past 1.75
    const int b = (int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u);
    return max(b, 0);
}

// Four codes of x * 2^(127 - b).
__device__ __forceinline__ uint32_t p8_codes(const float* x, int b) {
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        y[e] = __builtin_amdgcn_ldexpf(x[e], P8_ONE - b);
        // (of the last scale, the codes that stand for numbers of f32)
        if (b > P8_TOP && fabsf(y[e]) < __builtin_inff()) y[e] = fminf(fmaxf(y[e], -240.0f), 240.0f);
    }
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
}

// Four codes of scale byte `was` as codes of scale byte b >= was.
__device__ __forceinline__ uint32_t p8_again(uint32_t w, int was, int b) {
    const float x[4] = {__builtin_amdgcn_cvt_f32_fp8((int)w, 0), __builtin_amdgcn_cvt_f32_fp8((int)w, 1),
                        __builtin_amdgcn_cvt_f32_fp8((int)w, 2), __builtin_amdgcn_cvt_f32_fp8((int)w, 3)};
    return was == 255 ? 0x7f7f7f7fu : p8_codes(x, P8_ONE + b - was);
}

// A lane's part of a row's head: N dims of its lower half and those HD / 2 further (a
// rotation's pairs), of four lanes.
template <class T, int HD>
struct Append8Row {
    static constexpr int N = HD / 8, HALF = HD / 2;
    T lo[N], hi[N];
    float x[2][N];

    __device__ __forceinline__ void load(const T* from) {
        __builtin_memcpy(lo, __builtin_assume_aligned(from, 16), sizeof lo);
        __builtin_memcpy(hi, __builtin_assume_aligned(from + HALF, 16), sizeof hi);
    }
    // x, turned by the tables' rows from cs and sn on (null: as it is).
    __device__ __forceinline__ void turn(const float* cs, const float* sn) {
#pragma unroll
        for (int e = 0; e < N; e++) {
            x[0][e] = (float)lo[e];
            x[1][e] = (float)hi[e];
        }
        if (!cs) return;
        float cl[N], ch[N], sl[N], sh[N];
        __builtin_memcpy(cl, __builtin_assume_aligned(cs, 16), sizeof cl);
        __builtin_memcpy(ch, __builtin_assume_aligned(cs + HALF, 16), sizeof ch);
        __builtin_memcpy(sl, __builtin_assume_aligned(sn, 16), sizeof sl);
        __builtin_memcpy(sh, __builtin_assume_aligned(sn + HALF, 16), sizeof sh);
#pragma unroll
        for (int e = 0; e < N; e++) {
            const float y = x[0][e], w = x[1][e];
            x[0][e] = y * cl[e] - w * sl[e];
            x[1][e] = w * ch[e] + y * sh[e];
        }
    }
    // The largest finite magnitude.
    __device__ __forceinline__ float most() const {
        float a = 0.0f;
#pragma unroll
        for (int d = 0; d < 2; d++)
#pragma unroll
            for (int e = 0; e < N; e++) {
                const float y = fabsf(x[d][e]);
                a = y < __builtin_inff() ? fmaxf(a, y) : a;
            }
        return a;
    }
    __device__ __forceinline__ void put(uint8_t* to, int byte) const {
#pragma unroll
        for (int d = 0; d < 2; d++) {
            uint32_t w[N / 4];
#pragma unroll
            for (int e = 0; e < N / 4; e++) w[e] = p8_codes(x[d] + 4 * e, byte);
            __builtin_memcpy(__builtin_assume_aligned(to + d * HALF, 8), w, sizeof w);
        }
    }
    // Codes under byte `was` as codes under `byte`.
    __device__ __forceinline__ static void again(uint8_t* at, int was, int byte) {
#pragma unroll
        for (int d = 0; d < 2; d++) {
            uint32_t w[N / 4];
            __builtin_memcpy(w, __builtin_assume_aligned(at + d * HALF, 8), sizeof w);
#pragma unroll
            for (int e = 0; e < N / 4; e++) w[e] = p8_again(w[e], was, byte);
            __builtin_memcpy(__builtin_assume_aligned(at + d * HALF, 8), w, sizeof w);
        }
    }
};

// Workgroups below q_wgs: `parts` to a packed row, chunks of its q as paged_append_kernel
// takes them.  The others: a wavefront takes 16 rows of codes, four lanes a row,
//   NARROW      the same position of up to 16 heads of k and v, a row a wavefront: up to
//               A8_FEW new rows in a block are worked by the first one's, one after another,
//               the heads of more by all of them, each head's rows as below
//   otherwise   the up to 16 rows of a block, of one head of k or v
// Bound by HBM for many rows (11166 of f32, 32 heads over 8 of 128: 482 MB in 99 us,
// 4.9 TB/s, as a copy), by four memory round trips for few: the row's sequence (two),
// its page, its block's scale.
constexpr int A8_WG = 256, A8_FEW = 4, A8_SHORT = 3;
template <class T, int HD, bool NARROW>
__global__ __launch_bounds__(A8_WG) void paged8_append_kernel(PagedKv8 c, PagedRows b, int n_heads, int q_wgs, int parts,
                                                              const T* q, int ldq, const T* __restrict__ k, int ldk,
                                                              const T* __restrict__ v, int ldv,
                                                              const float* __restrict__ cs,
                                                              const float* __restrict__ sn, int rope_rows, T* q_out,
                                                              int ldqo) {
    constexpr int HALF = HD / 2;
    if ((int)blockIdx.x < q_wgs) {
        constexpr int CP = HALF / 8;
        const int row = (unsigned)blockIdx.x / (unsigned)parts, stride = A8_WG * parts;  // (a multiple of CP)
        int e = A8_WG * (blockIdx.x - row * parts) + threadIdx.x;
        const int i = 8 * (e % CP);
        T lo[8], hi[8];
        const auto fetch = [&] {  // (past the last head: the first one's again, not used)
            const T* x = q + (size_t)row * ldq + (e < CP * n_heads ? e / CP * HD : 0) + i;
            __builtin_memcpy(lo, __builtin_assume_aligned(x, 16), sizeof lo);
            __builtin_memcpy(hi, __builtin_assume_aligned(x + HALF, 16), sizeof hi);
        };
        fetch();
        const int s = pg_row_seq(b, row);
        if (s < 0) return;
        const PgSeq sq = pg_seq(b, s);
        if (row < sq.row0 || row >= sq.row0 + sq.n) return;
        const int pos = sq.kv - sq.n + (row - sq.row0);
        const bool bad = sq.bad || (cs && pos >= rope_rows), turned = cs && pos >= 0 && !bad;
        float cl[8], ch[8], sl[8], sh[8];
        if (turned) {
            const float *ct = cs + (size_t)pos * HD + i, *st = sn + (size_t)pos * HD + i;
            __builtin_memcpy(cl, __builtin_assume_aligned(ct, 16), sizeof cl);
            __builtin_memcpy(ch, __builtin_assume_aligned(ct + HALF, 16), sizeof ch);
            __builtin_memcpy(sl, __builtin_assume_aligned(st, 16), sizeof sl);
            __builtin_memcpy(sh, __builtin_assume_aligned(st + HALF, 16), sizeof sh);
        }
        for (; e < CP * n_heads; e += stride, fetch()) {
            T x[8], y[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                float u = (float)lo[j], w = (float)hi[j];
                if (turned) {
                    const float z = u;
                    u = z * cl[j] - w * sl[j];
                    w = w * ch[j] + z * sh[j];
                }
                x[j] = (T)(bad ? pg_nan() : pos < 0 ? 0.0f : u);
                y[j] = (T)(bad ? pg_nan() : pos < 0 ? 0.0f : w);
            }
            T* to = q_out + (size_t)row * ldqo + e / CP * HD + i;
            __builtin_memcpy(__builtin_assume_aligned(to, 16), x, sizeof x);
            __builtin_memcpy(__builtin_assume_aligned(to + HALF, 16), y, sizeof y);
        }
        return;
    }
    using R = Append8Row<T, HD>;
    const int lane = threadIdx.x & 63, sub = lane >> 2, i = R::N * (lane & 3);
    const int at = __builtin_amdgcn_readfirstlane((int)((blockIdx.x - q_wgs) * (A8_WG / 64) + (threadIdx.x >> 6)));
    // the positions of a sequence's rows that are stored
    const auto ends = [&](const PgSeq& x, int& first) {
        first = max(x.kv - x.n, 0);
        return x.n && !x.bad ? max(first, cs ? min(x.kv, rope_rows) : x.kv) : first;
    };
    int s, lo, hi;  // sequence, and the block's positions [lo, hi) that are new
    PgSeq sq;
    const auto row_of = [&](int pos, int head, bool value) {
        return (value ? v : k) + (size_t)(sq.row0 + pos - (sq.kv - sq.n)) * (value ? ldv : ldk) + head * HD + i;
    };
    const auto turn = [&](R& x, int pos, bool value) {
        const bool t = cs && !value;
        x.turn(t ? cs + (size_t)pos * HD + i : nullptr, sn + (t ? (size_t)pos * HD + i : 0));
    };
    // the block's first cache row of a head, from page 0's
    size_t row = 0;
    const auto find = [&] {
        bool none;
        const int j0 = lo & ~15, page = pg_page(c, b.table + (size_t)s * b.max_pages, j0, sq.kv, none);
        row = ((size_t)page * c.kv_heads << c.log_ps) + (j0 & ((1 << c.log_ps) - 1));
        return !none;
    };
    // the scale that rows of at most amax and older ones under `was` get
    const auto scale_of = [&](float amax, int was) {
        const int byte = p8_scale_of(amax);
        return lo & 15 && was != 255 ? max(was, byte) : byte;
    };
    // The block's rows of one head of k or v, four lanes a row.
    const auto by_rows = [&](int head, bool value) {
        const int j0 = lo & ~15, pos = j0 + sub;
        const bool mine = pos >= lo && pos < hi;
        const size_t at = row + ((size_t)head << c.log_ps);
        uint8_t* codes = static_cast<uint8_t*>(value ? c.v : c.k) + at * HD + i;
        uint8_t* scale = (value ? c.v_scale : c.k_scale) + (at >> 4);
        R x;
        x.load(row_of(mine ? pos : lo, head, value));
        const int was = lo > j0 ? *scale : 0;
        turn(x, mine ? pos : lo, value);
        float amax = x.most();  // (of the other lanes: lo's)
#pragma unroll
        for (int d = 1; d < 64; d *= 2) amax = fmaxf(amax, __shfl_xor(amax, d));
        const int byte = scale_of(amax, was);
        if (sub < lo - j0 && byte != was) R::again(codes + sub * HD, was, byte);
        if (mine) x.put(codes + sub * HD, byte);
        if (lane == 0) *scale = (uint8_t)byte;
    };
    if constexpr (NARROW) {
        const int waves = (2 * c.kv_heads + 15) >> 4, packed = (unsigned)at / (unsigned)waves;
        if (packed >= b.rows) return;
        const int unit0 = 16 * (at - packed * waves), unit = unit0 + sub;
        const bool mine = unit < 2 * c.kv_heads, value = unit >= c.kv_heads;
        const int head = mine ? unit - (value ? c.kv_heads : 0) : 0;
        R x;
        x.load((value ? v : k) + (size_t)packed * (value ? ldv : ldk) + head * HD + i);  // (most often the only row)
        s = pg_row_seq(b, packed);
        if (s < 0) return;
        sq = pg_seq(b, s);
        if (packed < sq.row0 || packed >= sq.row0 + sq.n) return;
        const int pos = sq.kv - sq.n + (packed - sq.row0);
        int first;
        const int end = ends(sq, first);
        if (pos < first || pos >= end) return;
        lo = max(pos & ~15, first);
        hi = min((pos | 15) + 1, end);
        if (hi - lo > A8_FEW) {
            // (row_start may decrease: rows of the block that are found in other sequences do no part)
            if (pg_row_seq(b, packed - (pos - lo)) != s) return;
            const bool all = pg_row_seq(b, packed + (hi - 1 - pos)) == s;
            if ((!all && pos != lo) || !find()) return;
            for (int u = unit0 + (all ? pos - lo : 0); u < min(unit0 + 16, 2 * c.kv_heads); u += all ? hi - lo : 1)
                by_rows(u < c.kv_heads ? u : u - c.kv_heads, u >= c.kv_heads);
            return;
        }
        if (pos != lo || !find()) return;
        const int j0 = lo & ~15;
        const size_t at0 = row + ((size_t)head << c.log_ps);
        uint8_t* codes = static_cast<uint8_t*>(value ? c.v : c.k) + at0 * HD + i;
        uint8_t* scale = (value ? c.v_scale : c.k_scale) + (at0 >> 4);
        const int was = lo > j0 ? *scale : 0;
        turn(x, lo, value);
        float amax = x.most();
        for (int p = lo + 1; p < hi; p++) {
            x.load(row_of(p, head, value));
            turn(x, p, value);
            amax = fmaxf(amax, x.most());
        }
        amax = fmaxf(amax, __shfl_xor(amax, 1));
        amax = fmaxf(amax, __shfl_xor(amax, 2));
        if (!mine) return;
        const int byte = scale_of(amax, was);
        if (byte != was)
            for (int r = 0; r < lo - j0; r++) R::again(codes + r * HD, was, byte);
        for (int p = hi - 1;; p--) {  // (the last one's is at hand)
            x.put(codes + (p - j0) * HD, byte);
            if (p == lo) break;
            x.load(row_of(p - 1, head, value));
            turn(x, p - 1, value);
        }
        if ((lane & 3) == 0) *scale = (uint8_t)byte;
    } else {
        const auto blocks = [&](const PgSeq& x) {
            int first;
            const int end = ends(x, first);
            return end > first ? ((end - 1) >> 4) - (first >> 4) + 1 : 0;
        };
        PgUnits<decltype(blocks)> pu(b, blocks);
        const int unit = (unsigned)at / (unsigned)(2 * c.kv_heads), of = at - unit * 2 * c.kv_heads;
        if (unit >= pu.total) return;
        int u, first;
        s = pu.find(unit, u);
        sq = pu.get(s);
        const int end = ends(sq, first), j = ((first >> 4) + u) << 4;
        lo = max(j, first);
        hi = min(j + 16, end);
        if (find()) by_rows(of >> 1, of & 1);
    }
}

// Few rows a sequence: NARROW.  us, NARROW / otherwise, 32 KV heads of 128, bf16 rows: 256
// sequences of one row 7.7 / 28, of three 13 / 29, 1024 of three 30 / 397, one of 256 beside
// 255 of one 10 / 29 (27 where all of a block's rows are worked by the first one's
// wavefront); but 64 of four 9.6 / 7.5, one of 500 11 / 7.5.
inline bool append8_narrow(const PagedRows& r) { return !r.row_start || r.rows <= (long)A8_SHORT * r.n_seqs; }

struct Append8Call {
    const PagedAppendArgs& p;
    const PagedKv8& c;
    hipStream_t s;
    template <class T, int HD>
    hipError_t run() const {
        const int chunks = HD / 16 * (p.q ? p.n_heads : 0);
        const int parts = chunks ? (chunks + A8_WG - 1) / A8_WG : 0;
        const long q_wgs = (long)p.rows.rows * parts, waves = paged8_append_waves(c, p.rows);
        const long wgs = q_wgs + (waves + A8_WG / 64 - 1) / (A8_WG / 64);
        const auto kernel = append8_narrow(p.rows) ? paged8_append_kernel<T, HD, true> : paged8_append_kernel<T, HD, false>;
        hipLaunchKernelGGL(kernel, dim3((unsigned)wgs), dim3(A8_WG), 0, s, c, p.rows, p.n_heads, (int)q_wgs, parts,
                           static_cast<const T*>(p.q), p.ldq, static_cast<const T*>(p.k), p.ldk,
                           static_cast<const T*>(p.v), p.ldv, p.cos, p.sin, p.rope_rows, static_cast<T*>(p.q_out),
                           p.ldqo);
        return hipGetLastError();
    }
};

}  // namespace

long paged8_append_waves(const PagedKv& kv, const PagedRows& r) {
    if (append8_narrow(r)) return (long)r.rows * ((2 * kv.kv_heads + 15) / 16);
    // n rows lie in at most n / 16 + 2 blocks of 16 positions
    return ((long)r.rows / 16 + 2l * (r.n_seqs < r.rows ? r.n_seqs : r.rows)) * 2 * kv.kv_heads;
}

hipError_t launch_paged8_append(int dtype, int hd, const PagedAppendArgs& p, const PagedKv8& c, hipStream_t s) {
    if (p.rows.rows <= 0 || p.rows.n_seqs <= 0) return hipSuccess;
    return paged8_with_types(dtype, hd, Append8Call{p, c, s});
}

size_t paged8_rows16_work_bytes(const PagedKv& kv, const PagedRows& r, int n_heads, int hd) {
    return rows16_work_bytes(kv, r, n_heads, hd, 1);
}

bool paged8_rows16_fits(const PagedKv& kv, const PagedRows& r, int n_heads, int hd) {
    return rows16_fits(kv, r, n_heads, hd, 1);
}

hipError_t launch_paged8_rows16(int dtype, int hd, const PagedAttendArgs& p, const PagedKv8& c, hipStream_t s) {
    if (p.rows.rows <= 0 || p.rows.n_seqs <= 0) return hipSuccess;
    return paged8_with_types(dtype, hd, Rows8Call{p, c, s});
}

}  // namespace frq
