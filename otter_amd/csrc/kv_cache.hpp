// The quantised K/V cache: layout, quantisation of one block, and which cache rows a call's rows are.
//
// A cache holds, for every episode and key head, `capacity` positions of head_dim numbers in blocks of 32 along the head
// dimension; a block is 32 codes (4-bit e2m1 or 8-bit e4m3) times one power of two.  With x the block's numbers and M the
// largest code (6 or 448):
//     e = the smallest integer in [-100, 100] with max|x| <= M 2^e (100 if there is none),   code = nearest(x / 2^e), ties to even,
// so x / 2^e is exact in fp32 and every stored number is exact in bf16 (at most 4 significant bits, exponents within fp32's):
// the attention multiplies the cache's numbers on bf16 matrix instructions without a rounding of its own.  The range of e keeps
// every non-zero number a normal one.  A block with a NaN or an infinity gets the scale byte 255 and reads back as NaN throughout.
// Writer, fused writer and reader share the hardware's block conversions (v_cvt_scalef32_*): round to nearest even; only the
// exponent field of their scale operand is used (checked on the device: sign and mantissa bits change nothing), 255 gives NaN.
#pragma once
#include "common.hpp"
#include "otter_hip.h"

struct KvGeom {
    unsigned char* codes;  long ckv, ce, ch;      // byte strides: keys -> values, episode, head (rows of RB bytes are contiguous)
    unsigned char* scales; long skv, se, sh;      // one 4-byte word per row: byte b = exponent of block b + 127
    int E, S, H;
    const int* idx;                               // [n] episode of row i; null: episode i
    const int* pos;                               // [E] window position of the row's first step; null: 0
    const int* count;                             // [n] steps of row i that exist; null: all
    int n, T;
};

struct KvRow { int e, pos, cnt; };                // e < 0: no such episode

__device__ __forceinline__ KvRow kv_row(const KvGeom& g, int i) {
    KvRow r;
    const int e = g.idx ? g.idx[i] : i;
    const bool ok = e >= 0 && e < g.E;
    r.e = ok ? e : -1;
    r.pos = (ok && g.pos) ? g.pos[e] : 0;
    r.pos = min(max(r.pos, -(1 << 30)), 1 << 30);                  // sums of a position and a step count stay in 32 bits
    r.cnt = g.count ? min(max(g.count[i], 0), g.T) : g.T;
    return r;
}

template <int BITS> struct KvFmt;
template <> struct KvFmt<4> {
    static constexpr unsigned kCarry = 0x3fffffu;                  // mantissas above 1.5 need the next exponent (6 = 1.5 * 2^2)
    static constexpr int kTop = 2;
    static constexpr float kMax = 6.0f;
};
template <> struct KvFmt<8> {
    static constexpr unsigned kCarry = 0x1fffffu;                  // 448 = 1.75 * 2^8
    static constexpr int kTop = 8;
    static constexpr float kMax = 448.0f;
};

// scale byte of a block whose largest magnitude has the bits `top`: the bit pattern of a non-negative float grows with its
// value and NaN's lies above infinity's, so one unsigned maximum finds the largest magnitude and any non-finite number
template <int BITS> __device__ __forceinline__ unsigned kv_scale_byte(unsigned top) {
    const int e = (int)((top + KvFmt<BITS>::kCarry) >> 23) - 127 - KvFmt<BITS>::kTop;
    return top >= 0x7f800000u ? 255u : (unsigned)(min(max(e, -100), 100) + 127);
}
__device__ __forceinline__ unsigned kv_abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// largest |x| (as bits) over the four lanes that hold one block of 32, eight numbers each
__device__ __forceinline__ unsigned kv_block_top(const float (&x)[8]) {
    unsigned t = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) t = max(t, kv_abs_bits(x[i]));
    t = max(t, (unsigned)__builtin_amdgcn_mov_dpp((int)t, 0xB1, 0xF, 0xF, true));      // quad_perm [1,0,3,2]
    return max(t, (unsigned)__builtin_amdgcn_mov_dpp((int)t, 0x4E, 0xF, 0xF, true));   // quad_perm [2,3,0,1]
}

// eight numbers -> codes (4-bit: one word, 8-bit: two), numbers in order from the lowest bits up
template <int BITS> __device__ __forceinline__ void kv_encode8(const float (&x)[8], unsigned scale_byte, unsigned (&w)[BITS / 4]) {
    const float sc = __uint_as_float(scale_byte << 23);
    const float lim = KvFmt<BITS>::kMax * sc;                       // only blocks past the largest exponent are cut (e4m3 has no infinity to overflow to)
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = __builtin_amdgcn_fmed3f(x[i], -lim, lim);
    if constexpr (BITS == 4) {
        unsigned r = 0;
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, y[0], y[1], sc, 0);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, y[2], y[3], sc, 1);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, y[4], y[5], sc, 2);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, y[6], y[7], sc, 3);
        w[0] = r;
    } else {
        typedef __attribute__((ext_vector_type(2))) short s16x2;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            s16x2 r = {0, 0};
            r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, y[4 * h], y[4 * h + 1], sc, false);
            r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, y[4 * h + 2], y[4 * h + 3], sc, true);
            w[h] = __builtin_bit_cast(unsigned, r);
        }
    }
}

// element type of k / v / q operands
template <typename T> struct KvElem;
template <> struct KvElem<float> { static constexpr int code = DT_F32; };
template <> struct KvElem<__bf16> { static constexpr int code = DT_BF16; };
template <> struct KvElem<_Float16> { static constexpr int code = DT_F16; };

// a result in the type of the activations; fp16: cut at its largest number (NaN stays), as everywhere in this library
template <typename T> __device__ __forceinline__ T kv_result(float v) {
    if constexpr (KvElem<T>::code == DT_F16) return (T)(v == v ? __builtin_amdgcn_fmed3f(v, -65504.f, 65504.f) : v);
    else return (T)v;
}

// eight consecutive numbers as they lie in memory; `vec`: 16-byte aligned
template <typename T> struct KvEight { typedef __attribute__((ext_vector_type(8))) T v8; };
template <typename T> __device__ __forceinline__ void kv_fetch8(const T* p, bool vec, typename KvEight<T>::v8& x) {
    if (vec) {
        x = *(const typename KvEight<T>::v8*)__builtin_assume_aligned(p, 16);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = p[i];
    }
}
// the same as floats
template <typename T> __device__ __forceinline__ void kv_load8(const T* p, bool vec, float (&x)[8]) {
    typename KvEight<T>::v8 r;
    kv_fetch8<T>(p, vec, r);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)r[i];
}

template <typename T> struct KvOperand { T* p; long row, step, head; };   // element strides

// host: checks of the C structs shared by every entry point; OTTER_OK or error set
int otter_kv_check(const otter_kv_cache* c, const otter_kv_rows* r, const char* name);
int otter_kv_check_writable(const otter_kv_cache* c, const char* name);
int otter_kv_check_operand(const otter_kv_operand* o, int dtype, bool write, const char* what, const char* name);
KvGeom otter_kv_geom(const otter_kv_cache* c, const otter_kv_rows* r);
