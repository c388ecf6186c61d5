// Causal attention of packed prompt rows over a paged KV cache (paged.hpp).
//
// A sequence's rows and the G = n_heads / kv_heads query heads of a KV head are
// one list of n * G query rows, as in paged.hip; a workgroup of four wavefronts
// takes 128 of them, 32 a wavefront, or 64, two wavefronts with half the keys each
// to 32 rows, and walks the keys in tiles of 64 that it stages in LDS: the next
// tile's LDS DMA runs while a tile is worked, one barrier a tile.
//   S^T (keys x rows) = K . Q^T on v_mfma_f32_32x32x16: the C layout leaves lane
//     32 h + n keys 8 i + 4 h + (0..3) of row n, which is what the second
//     product takes as its B operand, in a key order that V's reads follow: P
//     never moves between lanes.
//   O^T (dims x rows) += V^T . P^T: V^T comes out of the row-major V tile by the
//     transposing LDS read (ds_read_b64_tr_b16).
// LDS rows are kept unpadded (the DMA writes them in lane order); the DMA's
// source addresses permute the 16-byte chunks of a row instead, so that the
// rows one read touches fall in different banks.
// The running maximum is renewed only when a row's scores pass it by LAZY: the
// weights stay below 2^(SHIFT + LAZY) = 2^TOP, and the sums and the output share
// the factor whatever it is.  Of f16 parts it is also lowered where a
// tile's scores stay below it by PF_LOW (PG_DROP); tiles of 64 such rows of q and
// keys, N(0, 1), differ by less.
// 16-bit activations: p is rounded to the cache's type for the second product
// (a relative 2^-11 or 2^-8 of each weight at most, the output's own rounding;
// the sum l takes p as it is).  A second part, as the 16-row kernel keeps, costs
// half as many matrix instructions again, which are the bound here: a prompt of
// 16384 2.78 ms instead of 2.04, 17 ragged ones 0.196 instead of 0.159, for an
// output 0.0015 of it from 64 bits instead of 0.0020 (bf16; f16 0.0002, 0.0003).
// f32 activations: q and p in parts that keep f32's precision.
// One prompt of 16384, 32 heads over 8 of 128, bf16: 2.0 ms, 1.10 PFLOP/s, where a
// large matrix product of the library makes 1.19: the matrix pipe 57 % busy, beside
// 6.4 VALU instructions to an MFMA, at the 1.8 GHz that the chip's power leaves (the
// softmax left out: 2.03 of then 2.10 ms).  17 prompts of 67 .. 1683: 0.16 ms, 0.72
// PFLOP/s: some 9 key tiles to a tile of rows, whose start, masked last tile and end
// count, and 6 rounds of unequal workgroups.  No faster: two groups of wavefronts in
// turn at the matrix pipe, S^T of the next tile under this one's softmax, wave
// priorities, eight wavefronts on 256 rows, three tiles in LDS, three wavefronts a
// SIMD (spills).
#include <hip/hip_runtime.h>

#include "common.hpp"
#include "kernels.hpp"
#include "paged.hpp"

namespace frq {

namespace {

constexpr int PF_WAVES = 4;
constexpr int PF_ROWS = 32 * PF_WAVES;
constexpr int PF_KEYS = 64;
constexpr float PF_LOW = 8.0f;

typedef float pf_f16 __attribute__((ext_vector_type(16)));
typedef short pf_s4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ pf_f16 pf_mfma(PgElem<_Float16>::v8 a, PgElem<_Float16>::v8 b, pf_f16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ pf_f16 pf_mfma(PgElem<__bf16>::v8 a, PgElem<__bf16>::v8 b, pf_f16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// 64 lanes' 16 bytes from base + voff to LDS address lds + 16 * lane.  Written
// in assembly so that the compiler does not wait for it before every LDS read
// (it cannot tell the tile being filled from the one being read): the kernel
// waits itself.  One wait state between the M0 write and its use.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void pf_dma(const void* base, uint32_t voff, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(voff), "s"(base), "s"(lds)
                 : "memory", "m0");
}
#pragma clang diagnostic pop
__device__ __forceinline__ uint32_t pf_lds(const void* p) {
    return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t*)p;
}
__device__ __forceinline__ pf_s4 pf_read_tr(const uint8_t* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) pf_s4*)p);
}

__device__ __forceinline__ float pf_other_half(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __builtin_bit_cast(float, (threadIdx.x & 32) ? (uint32_t)a[0] : (uint32_t)a[1]);
}

template <class E, class T, int HD>
struct PrefillTile {
    using P = PgElem<E>;
    using v8 = typename P::v8;
    static constexpr bool WIDE = std::is_same<T, float>::value;
    static constexpr int NP = WIDE ? P::SPLIT : 1;
    static constexpr bool F16 = std::is_same<E, _Float16>::value;
    // (f16 parts of an f32 weight: as many of its digits as f16's range holds)
    static constexpr float LAZY = WIDE && F16 ? 0.0f : 7.0f, SHIFT = P::TOP - LAZY;
    static constexpr int KS = HD / 16, DT = HD / 32;   // steps of S^T, dim tiles of O^T
    static constexpr int ROW = 2 * HD, TILE = PF_KEYS * ROW;
    static constexpr int RPI = 512 / HD, NI = TILE / 1024;  // rows a DMA instruction, instructions a tile
    // LDS chunk pc of row r holds the row's chunk pc ^ kswz(r) of K, pc ^ vswz(r)
    // of V: the 16 rows by 16 bytes, and the 4 rows by 64, that a read touches at
    // once lie in different ones of the 64 banks.
    __device__ static __forceinline__ int kswz(int r) { return HD == 128 ? r & 15 : (r >> 1) & 7; }
    __device__ static __forceinline__ int vswz(int r) { return HD == 128 ? 4 * (r & 3) : 4 * ((r >> 1) & 1); }
};

// Whether KEYS rows of K and V from kt and vt on hold an infinite or NaN value, or
// a page of them is none.  Wave-uniform.
template <class X, class E, int KEYS>
__device__ __forceinline__ bool pf_odd(const uint8_t* kt, const uint8_t* vt, uint32_t bad) {
    bool any = bad & ((1u << KEYS / 16) - 1);
    for (int i = 16 * (threadIdx.x & 63); i < KEYS * X::ROW; i += 1024) {
        const pg_u4 k = *reinterpret_cast<const pg_u4*>(kt + i), v = *reinterpret_cast<const pg_u4*>(vt + i);
#pragma unroll
        for (int w = 0; w < 4; w++) any |= pg_word_odd<E>(k[w]) || pg_word_odd<E>(v[w]);
    }
    return __any(any);
}

// A workgroup takes one tile of query rows, or with CUT an equal contiguous
// range of all tiles' key tiles (head by head, sequence by sequence, tile by
// tile), as the 16-row kernel does: where a batch has fewer tiles than fill the
// chip and many keys each.  Tiles that a range cuts leave their sums in the
// workspace.
// KW wavefronts share 32 rows, with 64 / KW keys of a tile each.  KW = 2 is for
// batches of so few tiles that the one with the most keys lasts as long as the call:
// two of its workgroups, of 64 rows, work on a CU as one of 128 does, and end sooner
// where they are alone.  32 heads over 8, new rows 300 / 700 / 1000 (80 .. 256
// tiles), us: bf16 14.3 / 22.2 / 28.9 with KW = 1, 12.1 / 19.4 / 25.0 with 2, f32
// 18.0 / 29.1 / 39.2 and 14.4 / 24.2 / 32.5; beyond that not all of them start at
// once (1500 rows after 600, 384 tiles: 55 and 62).  (f32 rows over f16 pages take 4 %
// more on both sides since their maximum is renewed at every passing.)
constexpr int PF_FEW = 256;

template <class E, class T, int HD, int KW, bool CUT>
__global__ __launch_bounds__(64 * PF_WAVES, 2) void paged_prefill_kernel(PagedKv c, PagedRows b, int grp,
                                                                         const T* __restrict__ q, int ldq, float scale,
                                                                         T* __restrict__ out, int ldo,
                                                                         float* __restrict__ part,
                                                                         PgJoin* __restrict__ joins) {
    using X = PrefillTile<E, T, HD>;
    using v8 = typename X::v8;
    constexpr int RW = PF_WAVES / KW, ROWS = 32 * RW;
    constexpr int NA = 2 / KW;  // groups of 32 keys of a tile a wavefront
    __shared__ __align__(1024) uint8_t s_k[2][X::TILE], s_v[2][X::TILE];
    __shared__ float s_m[ROWS], s_l[ROWS];
    const int lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), w = KW == 1 ? wave : wave % RW;
    const int key0 = KW == 1 ? 0 : 32 * (wave / RW);  // first of its keys in a tile
    // key tiles of a sequence's tiles of rows (one where it has no keys)
    const auto key_tiles = [&](const PgSeq& x) { return x.kv <= PF_KEYS ? 1 : (x.kv + PF_KEYS - 1) / PF_KEYS; };
    const auto units = [&](const PgSeq& x) {
        const int row_tiles = (int)(((long)x.n * grp + ROWS - 1) / ROWS);
        return CUT ? row_tiles * key_tiles(x) : row_tiles;
    };
    PgUnits<decltype(units)> pu(b, units);
    int head, s, u;                       // KV head, sequence, unit of the sequence
    int at = 0, begin = 0, stop = 0, total = 0, n_wgs = 0, wg = 0;  // CUT: the range, and whose it is
    if constexpr (CUT) {
        total = pu.total * c.kv_heads;
        n_wgs = min((int)gridDim.x, total);
        // (each XCD takes a contiguous part of the list: a KV head's keys stay in one L2)
        wg = n_wgs % 8 == 0 && (int)blockIdx.x < n_wgs ? ((int)blockIdx.x & 7) * (n_wgs >> 3) + ((int)blockIdx.x >> 3)
                                                       : (int)blockIdx.x;
        if (wg >= n_wgs) {
            if (threadIdx.x == 0) joins[wg].rows = 0;
            return;
        }
        at = begin = pg_start(wg, total, n_wgs);
        stop = pg_start(wg + 1, total, n_wgs);
        head = (unsigned)begin / (unsigned)pu.total;
        s = pu.find(begin - head * pu.total, u);
    } else {
        // the last tiles of the sequences, which walk the most keys, first (sorted
        // over all sequences 3 % more: neighbours share a sequence's keys)
        head = blockIdx.x % c.kv_heads;
        const int unit = pu.total - 1 - (int)(blockIdx.x / c.kv_heads);
        if (unit < 0) return;
        s = pu.find(unit, u);
    }
    for (;;) {
        const PgSeq sq = pu.get(s);
        if constexpr (CUT) {
            if (sq.n == 0) {
                if (++s == b.n_seqs) {
                    s = 0;
                    head++;
                }
                continue;
            }
        }
        const int nk = CUT ? key_tiles(sq) : 1, tile = CUT ? (unsigned)u / (unsigned)nk : u;
        const int t0 = CUT ? u - tile * nk : 0, m_units = CUT ? min(nk - t0, stop - at) : 1;
        const bool whole = m_units == nk;
        const int rows = sq.n * grp, i0 = tile * ROWS;
        const int mine = min(i0 + 32 * w + n, rows - 1);
        const int row = sq.row0 + mine / grp, qh = head * grp + mine % grp;
        const int pos0 = sq.kv - sq.n;
        const int limit = pos0 + mine / grp;
        // last position of the workgroup's rows, first and last of this wavefront's
        const int wg_last = pos0 + min(i0 + ROWS - 1, rows - 1) / grp;
        const int first = pos0 + min(i0 + 32 * w, rows - 1) / grp;
        const int last = i0 + 32 * w < rows ? pos0 + min(i0 + 32 * w + 31, rows - 1) / grp : -1;
        int tiles = wg_last >= 0 ? wg_last / PF_KEYS + 1 : 0;
        if constexpr (CUT) tiles = min(tiles, t0 + m_units);

        pf_f16 o[X::DT];
        float m, l, peak;  // peak: the largest score so far

        // DMA: instruction i of this wavefront takes rows ((i PF_WAVES + wave) RPI) .. of
        // a tile, all in one group of 16 keys.  Source offsets of the lane within it:
        constexpr int CPR = HD / 8;
        const int dr = wave * X::RPI + lane / CPR, pc = lane % CPR;
        const uint32_t koff = (dr & 15) * X::ROW + 16 * (pc ^ X::kswz(dr));
        const uint32_t voff = (dr & 15) * X::ROW + 16 * (pc ^ X::vswz(dr));
        const int* table = b.table + (size_t)s * b.max_pages;
        // Byte offsets in the pools of 64 groups of 16 keys, lane i that of group i from
        // key id0 on, and which groups' page is none (theirs lead to page 0).
        int id0 = 0;
        uint32_t off_lo = 0, off_hi = 0;
        uint64_t none = 0;
        auto fetch_ids = [&](int j0) {
            id0 = j0;
            const int j = j0 + 16 * lane;
            bool off;
            const size_t page = pg_page(c, table, j, sq.kv, off);
            none = __ballot(off);
            const size_t at = (((page * c.kv_heads + head) << c.log_ps) + (j & ((1 << c.log_ps) - 1))) * X::ROW;
            off_lo = (uint32_t)at;
            off_hi = (uint32_t)(at >> 32);
        };
        auto issue = [&](int t) {
            const int j0 = t * PF_KEYS;
            if (j0 - id0 >= 1024) fetch_ids(j0);
            const int g0 = (j0 - id0) >> 4;
            const uint32_t kto = pf_lds(s_k[t & 1]) + wave * 1024, vto = pf_lds(s_v[t & 1]) + wave * 1024;
#pragma unroll
            for (int i = 0; i < X::NI / PF_WAVES; i++) {
                const int g = g0 + ((i * PF_WAVES + wave) * X::RPI >> 4);
                const uint64_t from = (uint64_t)(uint32_t)__builtin_amdgcn_readlane(off_hi, g) << 32 |
                                      (uint32_t)__builtin_amdgcn_readlane(off_lo, g);
                pf_dma(static_cast<const uint8_t*>(c.k) + from, koff, kto + i * PF_WAVES * 1024);
                pf_dma(static_cast<const uint8_t*>(c.v) + from, voff, vto + i * PF_WAVES * 1024);
            }
        };
        // LDS read offsets of this lane: K row n (+ 32), chunks 2 t + h; V rows
        // 4 h + (lane / 4) % 4 (+ 16 k + 8 j), dims 16 ((lane / 16) % 2) + 4 (lane % 4) (+ 32 d)
        const uint32_t kbase = n * X::ROW + 16 * (h ^ X::kswz(n));
        const int vr = (lane >> 2) & 3;
        const uint32_t vbase = (4 * h + vr) * X::ROW +
                               16 * ((2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) ^ X::vswz(vr)) + 8 * (lane & 1);

        if (t0 < tiles) {
            fetch_ids(t0 * PF_KEYS);
            issue(t0);
        }

        // Q^T, the B operand: dims 16 t + 8 h + e of row n (negated for a negative
        // scale: the maximum is taken of scores with a positive factor)
        v8 qf[X::NP][X::KS];
        float factor = fabsf(scale) * 1.4426950408889634f;
        const T* x = q + (size_t)row * ldq + (size_t)qh * HD + 8 * h;
        if constexpr (!X::WIDE) {
            const uint32_t flip = scale < 0.0f ? 0x80008000u : 0;
#pragma unroll
            for (int t = 0; t < X::KS; t++)
                qf[0][t] = __builtin_bit_cast(v8, *reinterpret_cast<const pg_u4*>(x + 16 * t) ^ flip);
        } else {
            float f[X::KS][8], a = 0.0f;
#pragma unroll
            for (int t = 0; t < X::KS; t++) {
                T raw[8];
                __builtin_memcpy(raw, __builtin_assume_aligned(x + 16 * t, 16), sizeof raw);
#pragma unroll
                for (int e = 0; e < 8; e++) f[t][e] = scale < 0.0f ? -raw[e] : raw[e];
            }
            if constexpr (std::is_same<E, _Float16>::value) {  // (parts of f16: scaled to the top of its range)
#pragma unroll
                for (int t = 0; t < X::KS; t++)
#pragma unroll
                    for (int e = 0; e < 8; e++) a = fmaxf(a, fabsf(f[t][e]));
                a = fmaxf(a, pf_other_half(a));
                const int ex = a > 0.0f && a < __builtin_inff() ? max(-100, __builtin_amdgcn_frexp_expf(a) - 15) : 0;
#pragma unroll
                for (int t = 0; t < X::KS; t++)
#pragma unroll
                    for (int e = 0; e < 8; e++) f[t][e] = __builtin_amdgcn_ldexpf(f[t][e], -ex);
                factor = __builtin_amdgcn_ldexpf(factor, ex);
            }
#pragma unroll
            for (int t = 0; t < X::KS; t++)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    float rest = f[t][e];
#pragma unroll
                    for (int p = 0; p < X::NP; p++) {
                        qf[p][t][e] = (E)rest;
                        rest -= (float)qf[p][t][e];
                    }
                }
        }

        const auto walk = [&](auto again) {
            constexpr bool AGAIN = decltype(again)::value;
#pragma unroll
            for (int d = 0; d < X::DT; d++)
#pragma unroll
                for (int i = 0; i < 16; i++) o[d][i] = 0.0f;
            m = peak = PG_LEAST;
            l = 0.0f;
            for (int t = t0; t < tiles; t++) {
                const int j0 = t * PF_KEYS;
                // tile t landed, in every wavefront, and tile t - 1 is read
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
                const uint32_t bad = (uint32_t)(none >> ((j0 - id0) >> 4)) & ((1u << PF_KEYS / 16) - 1);  // of its groups
                if (j0 + PF_KEYS > sq.kv || bad) {  // rows of V that are no keys hold anything
                    for (int ch = threadIdx.x; ch < X::TILE / 16; ch += 64 * PF_WAVES) {
                        const int r = ch / CPR;
                        if (j0 + r >= sq.kv || ((bad >> (r >> 4)) & 1))
                            reinterpret_cast<uint4*>(s_v[t & 1])[ch] = make_uint4(0, 0, 0, 0);
                    }
                    __syncthreads();
                }
                if (t + 1 < tiles) issue(t + 1);
                const int jw = j0 + key0;  // this wavefront's first key
                if (jw > last) continue;

                const uint8_t* kt = s_k[t & 1] + key0 * X::ROW;
                const uint8_t* vt = s_v[t & 1] + key0 * X::ROW;
                if (AGAIN && pf_odd<X, E, 64 / KW>(kt, vt, bad >> (key0 >> 4))) {
                    if (!__all(pg_all_nan(o)))
                        pg_plain<E, T, HD, 2>(
                            c, table, head, q + (size_t)row * ldq + (size_t)qh * HD, scale, limit, jw,
                            min(jw + 32 * NA, last + 1), X::SHIFT, h == 0, [&](int i) { return 8 * i + 4 * h; },
                            [&](int i, int e, float f, float p, float v) {
                                o[i / 4][4 * (i % 4) + e] = fmaf(p, v, o[i / 4][4 * (i % 4) + e] * f);
                            },
                            m, l);
                    peak = fmaxf(peak, m);
                    continue;
                }
                pf_f16 st[NA];
#pragma unroll
                for (int a = 0; a < NA; a++) {
#pragma unroll
                    for (int i = 0; i < 16; i++) st[a][i] = 0.0f;
#pragma unroll
                    for (int k = 0; k < X::KS; k++) {
                        const v8 kf = *reinterpret_cast<const v8*>(kt + 32 * a * X::ROW + (kbase ^ (32 * k)));
#pragma unroll
                        for (int p = X::NP - 1; p >= 0; p--) st[a] = pf_mfma(kf, qf[p][k], st[a]);
                    }
                }
                const bool mask = jw + 32 * NA - 1 > first || bad;
                if (mask) {
#pragma unroll
                    for (int a = 0; a < NA; a++)
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            const int r = 32 * a + (i & 3) + 8 * (i >> 2) + 4 * h;
                            if ((bad >> ((key0 + r) >> 4)) & 1) st[a][i] = pg_nan();
                            if (jw + r > limit) st[a][i] = -__builtin_inff();
                        }
                }
                float top = st[0][0];
#pragma unroll
                for (int a = 0; a < NA; a++)
#pragma unroll
                    for (int i = 0; i < 16; i++) top = fmaxf(top, st[a][i]);
                top = fmaxf(top, pf_other_half(top)) * factor;
                peak = fmaxf(peak, top);
                const float low = X::F16 ? fmaxf(top, peak - PG_DROP) : m;
                if (__any(top > m + X::LAZY || low < m - PF_LOW)) {
                    const float mn = fmaxf(top, low < m - PF_LOW ? low : m);
                    const float f = __builtin_amdgcn_exp2f(m - mn);  // (0 or 1 where nothing was seen before)
                    m = mn;
                    l *= f;
#pragma unroll
                    for (int d = 0; d < X::DT; d++) o[d] *= f;
                }
                // (fmaf: one operation less a weight.  Of scores past 2^30 it leaves what the
                // maximum was rounded by, which can be a weight that is infinite.)
                const float ms = m - X::SHIFT;
#pragma unroll
                for (int a = 0; a < NA; a++)
#pragma unroll
                    for (int i = 0; i < 16; i++) st[a][i] = AGAIN ? st[a][i] * factor - ms : fmaf(st[a][i], factor, -ms);
                if (mask) {  // (again: a factor of 0 would make NaN of -inf)
#pragma unroll
                    for (int a = 0; a < NA; a++)
#pragma unroll
                        for (int i = 0; i < 16; i++)
                            if (jw + 32 * a + (i & 3) + 8 * (i >> 2) + 4 * h > limit) st[a][i] = -__builtin_inff();
                }
                v8 pp[X::NP][2 * NA];
#pragma unroll
                for (int a = 0; a < NA; a++)
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        st[a][i] = __builtin_amdgcn_exp2f(st[a][i]);
                        l += st[a][i];
                        float rest = st[a][i];
#pragma unroll
                        for (int p = 0; p < X::NP; p++) {
                            pp[p][2 * a + (i >> 3)][i & 7] = (E)rest;
                            rest -= (float)pp[p][2 * a + (i >> 3)][i & 7];
                        }
                    }
#pragma unroll
                for (int k = 0; k < 2 * NA; k++)
#pragma unroll
                    for (int d = 0; d < X::DT; d++) {
                        const uint8_t* at = vt + 16 * k * X::ROW + (vbase ^ (64 * d));
                        const pf_s4 lo = pf_read_tr(at), hi = pf_read_tr(at + 8 * X::ROW);
                        const v8 vf = __builtin_bit_cast(v8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
                        for (int p = X::NP - 1; p >= 0; p--) o[d] = pf_mfma(vf, pp[p][k], o[d]);
                    }
            }
        };
        walk(std::false_type{});
        // Infinite or NaN sums: the same keys once more, tiles that hold such values
        // one key after another.  A prompt of 16384: 2.2 ms, with one infinite value 7.7,
        // all NaN 7.2, with one infinite value in every 16 keys, the worst there is, 205.
        if (__builtin_amdgcn_readfirstlane(__syncthreads_or(pg_odd(o)))) {
            fetch_ids(t0 * PF_KEYS);
            issue(t0);
            walk(std::true_type{});
        }
        l += pf_other_half(l);
        if constexpr (KW == 2) {  // the two that share rows
            static_assert(16 * X::DT * 64 * 4 * RW <= sizeof s_k, "the sums of half the wavefronts");
            __syncthreads();
            float* s_o = reinterpret_cast<float*>(s_k) + 16 * X::DT * 64 * w + lane;
            if (key0) {
#pragma unroll
                for (int d = 0; d < X::DT; d++)
#pragma unroll
                    for (int i = 0; i < 16; i++) s_o[64 * (16 * d + i)] = o[d][i];
                s_m[32 * w + n] = m;
                s_l[32 * w + n] = l;
            }
            __syncthreads();
            if (!key0) {
                const float m2 = s_m[32 * w + n], mn = fmaxf(m, m2);
                const float f = __builtin_amdgcn_exp2f(m - mn), f2 = __builtin_amdgcn_exp2f(m2 - mn);
                m = mn;
                l = l * f + s_l[32 * w + n] * f2;
#pragma unroll
                for (int d = 0; d < X::DT; d++)
#pragma unroll
                    for (int i = 0; i < 16; i++) o[d][i] = fmaf(s_o[64 * (16 * d + i)], f2, o[d][i] * f);
            }
        }
        if (key0 == 0 && i0 + 32 * w + n < rows) {
            if (!CUT || whole) {
                const float inv = sq.bad ? pg_nan() : limit < 0 ? 0.0f : 1.0f / l;  // (o is 0 in the first two)
                T* dst = out + (size_t)row * ldo + (size_t)qh * HD + 4 * h;
#pragma unroll
                for (int d = 0; d < X::DT; d++)
#pragma unroll
                    for (int g = 0; g < 4; g++) {
                        T y[4];
#pragma unroll
                        for (int i = 0; i < 4; i++) y[i] = (T)(o[d][4 * g + i] * inv);
                        __builtin_memcpy(__builtin_assume_aligned(dst + 32 * d + 8 * g, 8), y, sizeof y);
                    }
            } else {
                float* slot = part + ((size_t)2 * wg + (at != begin)) * pg_slot(ROWS, HD);
                float* dst = slot + (32 * w + n) * HD + 4 * h;
#pragma unroll
                for (int d = 0; d < X::DT; d++)
#pragma unroll
                    for (int g = 0; g < 4; g++)
                        *reinterpret_cast<pg_f4*>(dst + 32 * d + 8 * g) =
                            pg_f4{o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]};
                if (h == 0) {
                    slot[ROWS * HD + 32 * w + n] = m;
                    slot[ROWS * HD + ROWS + 32 * w + n] = l;
                }
            }
        }
        if constexpr (!CUT) return;
        if (at + m_units == stop) {
            if (threadIdx.x == 0)
                joins[wg] = pg_join(t0 == 0 && !whole, min(ROWS, rows - i0), sq, head, i0, at + nk - 1, total, n_wgs,
                                    2 * wg + (at != begin));
            return;
        }
        at += m_units;
        u += m_units;
        if (u == (int)(((long)rows + ROWS - 1) / ROWS) * nk) {
            u = 0;
            if (++s == b.n_seqs) {
                s = 0;
                head++;
            }
        }
        __syncthreads();  // the last key tile is read
    }
}

struct PrefillCall {
    const PagedAttendArgs& p;
    hipStream_t s;
    template <class E, class T, int HD>
    hipError_t run() const {
        const int grp = p.n_heads / p.kv.kv_heads;
        const T* q = static_cast<const T*>(p.q);
        T* out = static_cast<T*>(p.out);
        const long tiles = pg_tiles_bound(p.rows, grp, PF_ROWS) * p.kv.kv_heads;
        if (pg_kind(p.kv, p.rows, p.n_heads, HD) != PG_CUT) {
            const bool few = tiles <= PF_FEW;
            const auto kernel =
                few ? paged_prefill_kernel<E, T, HD, 2, false> : paged_prefill_kernel<E, T, HD, 1, false>;
            const long wgs = few ? pg_tiles_bound(p.rows, grp, PF_ROWS / 2) * p.kv.kv_heads : tiles;
            hipLaunchKernelGGL(kernel, dim3((unsigned)wgs), dim3(64 * PF_WAVES), 0, s, p.kv, p.rows, grp, q, p.ldq,
                               p.scale, out, p.ldo, nullptr, nullptr);
            return hipGetLastError();
        }
        float* part = static_cast<float*>(p.work);
        PgJoin* joins = reinterpret_cast<PgJoin*>(part + (size_t)2 * PG_WGS * pg_slot(PF_ROWS, HD));
        hipLaunchKernelGGL((paged_prefill_kernel<E, T, HD, 1, true>), dim3(PG_WGS), dim3(64 * PF_WAVES), 0, s, p.kv,
                           p.rows, grp, q, p.ldq, p.scale, out, p.ldo, part, joins);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        return launch_paged_join(dtype_of<T>(), HD, joins, part, PG_WGS, tiles, PF_ROWS, PF_ROWS, grp, p.out, p.ldo, s);
    }
    template <class T>
    static int dtype_of() {
        return std::is_same<T, float>::value ? GGML_F32 : std::is_same<T, _Float16>::value ? GGML_F16 : GGML_BF16;
    }
};

}  // namespace

bool paged_prefill_fits(const PagedKv& kv, const PagedRows& r, int n_heads) {
    return pg_tiles_bound(r, n_heads / kv.kv_heads, PF_ROWS) * kv.kv_heads <= PG_GRID;
}

size_t paged_prefill_work_bytes(const PagedKv& kv, const PagedRows& r, int n_heads, int hd) {
    if (pg_kind(kv, r, n_heads, hd) != PG_CUT) return 0;
    return PG_WGS * (2 * pg_slot(PF_ROWS, hd) * sizeof(float) + sizeof(PgJoin));
}

hipError_t launch_paged_prefill(int kv_dtype, int dtype, int hd, const PagedAttendArgs& p, hipStream_t s) {
    if (p.rows.rows <= 0 || p.rows.n_seqs <= 0) return hipSuccess;
    return paged_with_types(kv_dtype, dtype, hd, PrefillCall{p, s});
}

}  // namespace frq
