// The 8-bit paged KV cache: its view and what its kernels share (paged8.hip,
// paged_prefill.hip).
//
// Cache: k and v are [n_pages][kv_heads][page_size][HD] e4m3 codes (OCP: a sign,
// four bits of exponent, three of mantissa; largest 448, no infinities, 0x7f and 0xff
// NaN); k_scale and v_scale [n_pages][kv_heads][page_size / 16] bytes b, a scale of
// 2^(b - 127) (255: NaN) for the 16 rows of a head from a multiple of 16 on:
//   value = code * 2^(b - 127)
// A power of two takes nothing from the codes' digits: a code times its scale is a
// bf16 number, so the attention is that of a bf16 cache behind other loads, and
// codes under a grown scale are the old ones with another exponent.
#pragma once

#include "paged.hpp"

namespace frq {

struct PagedKv8 : PagedKv {
    uint8_t* k_scale;
    uint8_t* v_scale;
};

// Positions of a head that share a scale.
constexpr int P8_BLOCK = 16;
// Scale bytes of 2^0, and above which 448 codes leave f32's range.
constexpr int P8_ONE = 127, P8_TOP = 127 + 119;

#ifdef __HIPCC__

// The scale of byte b as an f32 factor, and as the operand of a scaled conversion
// (which takes its exponent alone, 255 for NaN).
__device__ __forceinline__ float p8_factor(int b) {
    return b == 255 ? pg_nan() : __builtin_bit_cast(float, b ? b << 23 : 1 << 22);
}
__device__ __forceinline__ float p8_operand(int b) { return __builtin_bit_cast(float, b << 23); }

// Two codes of a word, its high or low half, as they are or as values.
template <bool HI>
__device__ __forceinline__ uint32_t p8_pair(uint32_t w, float operand, __bf16) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, operand, HI));
}
template <bool HI>
__device__ __forceinline__ uint32_t p8_pair(uint32_t w, float operand, _Float16) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, operand, HI));
}
// Eight of them as the operand of a product.
template <class E>
__device__ __forceinline__ typename PgElem<E>::v8 p8_eight(uint32_t a, uint32_t b, float operand) {
    const pg_u4 w{p8_pair<false>(a, operand, E()), p8_pair<true>(a, operand, E()), p8_pair<false>(b, operand, E()),
                  p8_pair<true>(b, operand, E())};
    return __builtin_bit_cast(typename PgElem<E>::v8, w);
}

// Byte `at` of a pool, in scalar registers: loads from there take 32-bit offsets of the
// lanes.  (Left to itself the compiler adds pool, group and lane in vector registers.)
template <class T>
using P8Global = __attribute__((address_space(1))) T;
__device__ __forceinline__ const P8Global<uint8_t>* p8_base(const void* pool, uint64_t at) {
    uint64_t u = (uint64_t)pool + at;
    asm("" : "+s"(u));
    return (const P8Global<uint8_t>*)u;
}

// Whether a word holds a NaN code.
__device__ __forceinline__ bool p8_word_nan(uint32_t w) {
    const uint32_t t = ~(w | 0x80808080u);  // a zero byte where there is one
    return ((t - 0x01010101u) & ~t & 0x80808080u) != 0;
}

// 64 groups of 16 keys, lane i the one at position j0 + 16 i: where its rows are in
// the pools, its scales, and which groups' page is none (those and the ones behind
// the sequence's end lead to page 0).  Keys whose codes may stand for more than f32
// holds have a NaN scale here: products with their codes do not make infinities of
// them, and what is NaN is taken key by key, as it is.
struct P8Groups {
    uint32_t off_lo, off_hi;
    int k_scale, v_scale;
    uint64_t none;

    template <int HD>
    __device__ __forceinline__ void load(const PagedKv8& c, const int* table, int head, int j0, int kv) {
        const int j = j0 + 16 * (int)(threadIdx.x & 63), in = j & ((1 << c.log_ps) - 1);
        bool off;
        const size_t page = pg_page(c, table, j, kv, off);
        none = __ballot(off);
        const size_t row = ((page * c.kv_heads + head) << c.log_ps) + in;
        k_scale = c.k_scale[row >> 4];
        if (k_scale > P8_TOP) k_scale = 255;
        v_scale = c.v_scale[row >> 4];
        off_lo = (uint32_t)(row * HD);
        off_hi = (uint32_t)(row * HD >> 32);
    }
    // Of group g, wave-uniform.
    __device__ __forceinline__ uint64_t at(int g) const {
        return (uint64_t)(uint32_t)__builtin_amdgcn_readlane(off_hi, g) << 32 |
               (uint32_t)__builtin_amdgcn_readlane(off_lo, g);
    }
};

// PgCells of this cache.
template <int HD>
struct P8Cells {
    const uint8_t *k, *v;
    float ks, vs;
    __device__ __forceinline__ P8Cells(const PagedKv8& c, int page, int head, int j) {
        const size_t row = ((((size_t)page * c.kv_heads + head) << c.log_ps) + (j & ((1 << c.log_ps) - 1)));
        k = static_cast<const uint8_t*>(c.k) + row * HD;
        v = static_cast<const uint8_t*>(c.v) + row * HD;
        ks = p8_factor(c.k_scale[row >> 4]);
        vs = p8_factor(c.v_scale[row >> 4]);
    }
    __device__ __forceinline__ static void read(const uint8_t* at, float s, float (&x)[4]) {
        const int w = *reinterpret_cast<const int*>(at);
        x[0] = __builtin_amdgcn_cvt_f32_fp8(w, 0) * s;
        x[1] = __builtin_amdgcn_cvt_f32_fp8(w, 1) * s;
        x[2] = __builtin_amdgcn_cvt_f32_fp8(w, 2) * s;
        x[3] = __builtin_amdgcn_cvt_f32_fp8(w, 3) * s;
    }
    __device__ __forceinline__ void key(int u, int d, float (&x)[4]) const { read(k + u * HD + d, ks, x); }
    __device__ __forceinline__ void value(int u, int d, float (&x)[4]) const { read(v + u * HD + d, vs, x); }
};

// Calls f.run<T, HD>() for the types of a call.
template <class F>
hipError_t paged8_with_types(int dtype, int hd, F f) {
    const bool h64 = hd == 64;
    if (dtype == GGML_F32) return h64 ? f.template run<float, 64>() : f.template run<float, 128>();
    if (dtype == GGML_F16) return h64 ? f.template run<_Float16, 64>() : f.template run<_Float16, 128>();
    if (dtype == GGML_BF16) return h64 ? f.template run<__bf16, 64>() : f.template run<__bf16, 128>();
    return hipErrorInvalidValue;
}

#endif  // __HIPCC__

}  // namespace frq
