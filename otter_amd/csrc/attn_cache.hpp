// Attention over the quantised K/V cache (kv_cache.hpp): flash form, one or many new positions a row, grouped heads.
//
//   out[t, h] = sum_j p_j v_j / sum_j p_j,   p_j = 2^(c (q . k_j) - m),   c = scale log2 e,   m = running maximum of c (q . k_j),
// over the cached positions j that query t of the row sees.
//
// Operands.  A stored number has at most 4 significant bits, so k_j and v_j are exact in bf16 and the products run on
// v_mfma_f32_16x16x32_bf16 with fp32 accumulation.  q and p are written as sums of bf16 terms: q exactly (1 term for bf16, 2 for
// fp16, 3 for fp32), p in 2 terms (2^-16 relative, far below the output's own rounding) for 16-bit and 3 (2^-24) for fp32 outputs.
//
// For 16-bit activations and many columns the second product runs on fp16 operands instead, as long as the values allow it (see
// `Products`): one fp16 term is off by at most 2^-11 of a weight (an eighth of a bf16 output's own half step, 2^-8; numerator and
// denominator take the same rounded weight), so bf16 outputs need one term where bf16 weights need two; fp16 outputs take two, 2^-22.
// With one term 8 % of bf16 outputs are the neighbour of the rounded result, with two 0.04 %; the error against 64 bits is 1.6e-3 of the norm
// with either, that of the output's rounding.  The second term costs 124 against 107 us (8 windows of 2047) and 472 against 397 (500-step
// chunk).  A caller that wants every bit passes fp32 activations (2^-24 throughout).
//
// Tile.  A wave owns 16 * QT columns (query positions x heads of one key head's group) and walks over tiles of 32 keys, all
// state in registers.  S^T = K Q^T puts 8 scores of one column in a lane, keys 4g+i and 16+4g+i (g = lane / 16), which is the
// B operand of out^T = V^T P^T if V's rows are taken in the same key order: no exchange between lanes.  K is loaded as it lies
// (lane = key, head_dim / 4 consecutive numbers), V as 8 rows x head_dim / 16 numbers a lane and turned by v_perm after the
// conversion.  Rows past the last key are never read (addresses are cut at it).
//
// Masked keys.  Scores are selected, but 0 * NaN of a masked value row would still reach the accumulator.  Only tiles at the end of
// somebody's range have masked keys; where such a tile holds a scale byte that may stand for a non-finite block (>= 224; the
// writer's finite ones end at 227) its value rows are cleaned before the product, and the column is marked if it really sees
// one of them.  A lane's accumulators lie in one block of 32, so one mark a column is enough.
#pragma once
#include "kv_cache.hpp"

struct AttnCacheArgs {
    KvGeom g;
    KvOperand<const void> q; int q_vec;
    KvOperand<void> out;
    KvOperand<const void> kn, vn; int new_vec;      // fresh key / value rows to append (null: the cache is complete)
    int G, N, CG;                                   // query heads per key head, columns T * G, column groups of 16 * QT (64 * QT: wide)
    int causal, window, max_len;
    float c;
    int vec;                                        // 1: one step, one or two columns, on the vector unit
    int wide;                                       // 1: four waves x 16 QT columns a workgroup over tiles that they convert together
    int longest;                                    // wide: 1: (row, column group) pairs in order of their work (causal, no window, at most 64 rows)
    int kw, nsplit, chunk;                          // waves per item along the keys (1 or 4), splits of the key range, keys per split (multiple of 32 * kw)
    float* part;                                    // [nsplit][n * H][N][D + 2] partial sums: D numbers, maximum, sum
};

// positions that the columns [c0, c1] of a row look at: [beg, end); also the last position that all of them see and the first
struct KeyRange { int beg, end, hi_all, lo_all; };
__device__ __forceinline__ KeyRange key_range(const AttnCacheArgs& a, const KvRow& r, int c0, int c1) {
    KeyRange k{0, 0, -1, 0};
    const int t0 = c0 / a.G, t1 = min(c1 / a.G, r.cnt - 1);
    if (r.e < 0 || t0 > t1) return k;
    const int cap = min(a.g.S, a.max_len);
    const int q0 = a.causal ? r.pos + t0 : r.pos + r.cnt - 1, q1 = a.causal ? r.pos + t1 : q0;
    k.end = max(min(q1 + 1, cap), 0);
    k.beg = a.window ? max(q0 - a.window + 1, 0) : 0;
    k.hi_all = min(q0, cap - 1);
    k.lo_all = a.window ? max(q1 - a.window + 1, 0) : 0;
    k.beg = min(k.beg, k.end);
    return k;
}

template <typename T> struct AttnTerms;
template <> struct AttnTerms<__bf16> { static constexpr int q = 1, p = 2; };
template <> struct AttnTerms<_Float16> { static constexpr int q = 2, p = 2; };
template <> struct AttnTerms<float> { static constexpr int q = 3, p = 3; };

// Operand types and terms of the two products.  HALF: the values (and, for fp16 activations, the keys: the query is then one exact
// term) as fp16.  A block's numbers are exact in fp16 if its exponent e leaves them between 2^-24 and 65504: -23 <= e <= 13 for
// e2m1 (blocks whose largest number is between 1e-6 and 5e4).  e4m3 has a range of its own, so its numbers are taken 2^kUp times as large:
// -20 <= e <= 2, largest numbers between 4e-4 and 1.8e3, where -15 <= e would send any key whose values are below 7e-3 the long
// way (8 windows of 2047 steps, 12 heads of 64 with such keys: fp16 281 us, bf16 215; now 136 and 108).
// A workgroup that meets any other block that holds numbers starts over in bf16 terms (a block of zeros has the lowest exponent, -100: where
// scale bytes below the range were met, the codes decide).  Weights are scaled by 2^11 (below 2^15 with the reference's growth of 2^4): the smallest fp16 number is then 2^-35
// of the largest weight.
template <int BITS> constexpr int kUp = BITS == 8 ? 5 : 0;
template <typename T, bool HALF> struct Products { typedef __bf16 key, value; static constexpr int q = AttnTerms<T>::q, p = AttnTerms<T>::p; static constexpr float growth = 8.f, lift = 0.f; };
template <> struct Products<__bf16, true> { typedef __bf16 key; typedef _Float16 value; static constexpr int q = 1, p = 1; static constexpr float growth = 4.f, lift = 11.f; };
template <> struct Products<_Float16, true> { typedef _Float16 key, value; static constexpr int q = 1, p = 2; static constexpr float growth = 4.f, lift = 11.f; };

// With one term a weight its sum is one more product, with a row of ones: 16 matrix cycles for 8 weights a lane where additions take 32.
template <typename T, bool HALF> constexpr bool kSumByProduct = HALF && Products<T, HALF>::p == 1;

// most columns (in units of 16) that a wave of the wide form takes.  Each tile's operands are read from the LDS once for all of
// them, so 32 are faster wherever their accumulators leave room for the queries' terms: 8 windows of 2047 steps, 12 heads of 64,
// fp16 136 us against 148 with 16.  fp32 queries are three terms: 174 with 16 against 218 with 32 (spilled); so are 96 or 128
// numbers a head of fp16.
constexpr int wide_columns(int dtype, int nb) { return dtype == DT_BF16 || (dtype == DT_F16 && nb <= 2) ? 2 : 1; }

// the same of the narrow form: the three terms of fp32 queries leave no room for 32 with 96 or 128 numbers a head (300 rows x 8 heads
// of 96 x 32 steps over 300 positions 61 us with 16, 83 with 32; 8 heads of 64 over 1000: 115 and 97)
constexpr int narrow_columns(int dtype, int nb) { return dtype == DT_F32 && nb > 2 ? 1 : 2; }

// workgroups of the narrow form that a compute unit holds (waves a SIMD): fp32 heads of 128 do not fit the registers of three (one
// position, 64 rows x 32 / 8 heads over 4096: 69 us with two, 98 with three; heads of 96 fit: 62 with either, 300 x 32 steps 60 against 81)
constexpr int narrow_groups(int dtype, int nb, int qt) { return qt > 1 || (dtype == DT_F32 && nb == 4) ? 2 : 3; }

// host: instantiated per element type (attn_cache_*.hip)
template <typename T> int otter_attn_cache_launch(const AttnCacheArgs& a, int nb, int bits, int qt, unsigned blocks, hipStream_t s);

#ifdef OTTER_ATTN_CACHE_IMPL
namespace {

typedef __attribute__((ext_vector_type(4))) unsigned u32x4;

// what one tile of 32 keys needs from memory, as loaded
template <int NB, int BITS> struct RawTile {
    static constexpr int KW = NB * BITS / 4;                       // words of one key a lane holds (a quarter of its row)
    static constexpr int DV = NB == 3 ? 8 : 2 * NB;                // numbers of a value row a lane holds (NB = 3: 12 of 16 lanes, 8 each)
    static constexpr int VW = DV * BITS / 8 > 4 ? 2 : 1;           // words of those
    unsigned k[2][KW], v[8][VW];
    unsigned ks[2], vs[8];                                         // scale words of the rows
};

struct TileSource { const unsigned char* k; const unsigned char* v; const unsigned char* ks; const unsigned char* vs; };   // rows and scale words of this episode and head

__device__ __forceinline__ int v_row(int g, int i) { return 4 * g + (i & 3) + 16 * (i >> 2); }   // key of element i of lane group g's operand

// Rows are read through buffer resources that end with the tile's last existing row: what lies behind reads as zeros (checked
// word by word; scale byte 0 with codes 0 is the number 0), so a ragged tile needs no addresses of its own, and every load is a
// 32-bit lane offset from a scalar base.
template <int MOST = 32> __device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_of(const unsigned char* base, int k0, int row_bytes, int rows) {
    const unsigned long long at = (unsigned long long)base + (unsigned long long)k0 * row_bytes;
    const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)at), hi = __builtin_amdgcn_readfirstlane((unsigned)(at >> 32));
    return __builtin_amdgcn_make_buffer_rsrc((void*)(((unsigned long long)hi << 32) | lo), 0, __builtin_amdgcn_readfirstlane(min(max(rows, 0), MOST) * row_bytes), 0x00027000);   // no rows: everything reads as zeros
}
template <int BYTES, int W> __device__ __forceinline__ void buffer_words(__amdgpu_buffer_rsrc_t r, int off, unsigned (&w)[W]) {
    if constexpr (BYTES == 1) w[0] = __builtin_amdgcn_raw_buffer_load_b8(r, off, 0, 0);
    else if constexpr (BYTES == 2) w[0] = __builtin_amdgcn_raw_buffer_load_b16(r, off, 0, 0);
    else if constexpr (BYTES == 4) w[0] = __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0);
    else if constexpr (BYTES == 8 || BYTES == 24) {
#pragma unroll
        for (int i = 0; i < W; i += 2) { const auto u = __builtin_amdgcn_raw_buffer_load_b64(r, off + 4 * i, 0, 0); w[i] = u[0]; w[i + 1] = u[1]; }
    } else if constexpr (BYTES == 12) {
        const auto u = __builtin_amdgcn_raw_buffer_load_b96(r, off, 0, 0);
        w[0] = u[0]; w[1] = u[1]; w[2] = u[2];
    } else {
#pragma unroll
        for (int i = 0; i < W; i += 4) {
            const auto u = __builtin_amdgcn_raw_buffer_load_b128(r, off + 4 * i, 0, 0);
            w[i] = u[0]; w[i + 1] = u[1]; w[i + 2] = u[2]; w[i + 3] = u[3];
        }
    }
}

// key (value) rows k0 .. k0 + 31 of the cache, of which the first `rows` exist
template <int NB, int BITS> __device__ __forceinline__ void load_keys(RawTile<NB, BITS>& r, const TileSource& src, int k0, int rows, int lane) {
    constexpr int RB = 4 * NB * BITS, KB = RB / 4;
    const int li = lane & 15, g = lane >> 4;
    const auto kc = rows_of(src.k, k0, RB, rows), ks = rows_of(src.ks, k0, 4, rows);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        buffer_words<KB>(kc, li * RB + g * KB + 16 * h * RB, r.k[h]);
        r.ks[h] = __builtin_amdgcn_raw_buffer_load_b32(ks, li * 4 + 64 * h, 0, 0);
    }
}
template <int NB, int BITS> __device__ __forceinline__ void load_values(RawTile<NB, BITS>& r, const TileSource& src, int k0, int rows, int lane) {
    constexpr int RB = 4 * NB * BITS, DV = RawTile<NB, BITS>::DV, VB = DV * BITS / 8;
    const int li = lane & 15, g = lane >> 4;
    const auto vc = rows_of(src.v, k0, RB, rows), vs = rows_of(src.vs, k0, 4, rows);
    int vl = (NB == 3 ? min(li, 11) : li) * VB + 4 * g * RB;       // NB = 3: lanes 12 .. 15 repeat lane 11 (their output rows are not stored)
    asm("" : "+v"(vl));                                            // (a sum, not an `or`, of it and a constant goes into the load instruction)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const auto u = __builtin_amdgcn_raw_buffer_load_b128(vs, 16 * g + 64 * h, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) r.vs[4 * h + i] = u[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) buffer_words<VB>(vc, vl + ((i & 3) + 16 * (i >> 2)) * RB, r.v[i]);
}
template <int BYTES, int W> __device__ __forceinline__ void lds_words(const unsigned char* p, unsigned (&w)[W]) {
    if constexpr (BYTES == 1) w[0] = *p;
    else if constexpr (BYTES == 2) w[0] = *(const unsigned short*)p;
    else {
#pragma unroll
        for (int i = 0; i < W; ++i) w[i] = *(const unsigned*)(p + 4 * i);
    }
}

// scale operand of a block conversion: the wanted byte moved to the exponent's place (the conversion reads nothing else)
__device__ __forceinline__ float scale_of(unsigned word, int block) {
    const unsigned rot = (unsigned)(9 + 8 * block) & 31u;         // rotate right by 9 + 8 b: byte b lands on bits 23 .. 30
    return __uint_as_float(__builtin_amdgcn_alignbit(word, word, rot));
}
// the same times 2^UP; the addition stops at the byte 255, which says that the block is no number
template <int UP> __device__ __forceinline__ float scale_up(unsigned word, int block) {
    if constexpr (UP == 0) return scale_of(word, block);
    const unsigned rot = (unsigned)(8 + 8 * block) & 31u;         // byte b on bits 24 .. 31
    return __uint_as_float(__builtin_elementwise_add_sat(__builtin_amdgcn_alignbit(word, word, rot), (unsigned)UP << 24) >> 1);
}

// pair number j of a lane's words as two numbers of type V
template <int BITS, typename V = __bf16> __device__ __forceinline__ unsigned decode_pair(const unsigned* w, int j, float sc) {
    if constexpr (sizeof(V) == 2 && KvElem<V>::code == DT_F16) {
        f16x2 d;
        if constexpr (BITS == 4) {
            if (j % 4 == 0) d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w[j / 4], sc, 0);
            else if (j % 4 == 1) d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w[j / 4], sc, 1);
            else if (j % 4 == 2) d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w[j / 4], sc, 2);
            else d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w[j / 4], sc, 3);
        } else {
            if (j & 1) d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[j >> 1], sc, true);
            else d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[j >> 1], sc, false);
        }
        return __builtin_bit_cast(unsigned, d);
    } else {
        bf16x2 d;
        if constexpr (BITS == 4) {
            if (j % 4 == 0) d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[j / 4], sc, 0);
            else if (j % 4 == 1) d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[j / 4], sc, 1);
            else if (j % 4 == 2) d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[j / 4], sc, 2);
            else d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[j / 4], sc, 3);
        } else {
            if (j & 1) d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[j >> 1], sc, true);
            else d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[j >> 1], sc, false);
        }
        return __builtin_bit_cast(unsigned, d);
    }
}
// eight consecutive codes (from word w of a lane's row part on)
template <int BITS, typename V = __bf16> __device__ __forceinline__ typename Half16<V>::v8 decode8(const unsigned* w, float sc) {
    const u32x4 d = {decode_pair<BITS, V>(w, 0, sc), decode_pair<BITS, V>(w, 1, sc), decode_pair<BITS, V>(w, 2, sc), decode_pair<BITS, V>(w, 3, sc)};
    return __builtin_bit_cast(typename Half16<V>::v8, d);
}

__device__ __forceinline__ unsigned pack_bf16(float a, float b) {
    return __builtin_bit_cast(unsigned, (bf16x2){(__bf16)a, (__bf16)b});
}

// eight numbers as NP operands of type V whose sum they are (to the rounding of the last term)
template <int NP, typename V = __bf16> __device__ __forceinline__ void split_p(const float (&p)[8], typename Half16<V>::v8 (&out)[NP]) {
    unsigned w[NP][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float a = p[2 * i], b = p[2 * i + 1];
#pragma unroll
        for (int n = 0; n < NP; ++n) {
            if constexpr (KvElem<V>::code == DT_F16) {
                w[n][i] = __builtin_bit_cast(unsigned, (f16x2){(_Float16)a, (_Float16)b});
                if (n + 1 < NP) {                                  // (one instruction a rest: mixed precision takes either half as it lies)
                    asm("v_fma_mix_f32 %0, %1, -1.0, %0 op_sel_hi:[1,0,0]" : "+v"(a) : "v"(w[n][i]));
                    asm("v_fma_mix_f32 %0, %1, -1.0, %0 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "+v"(b) : "v"(w[n][i]));
                }
            } else {
                w[n][i] = pack_bf16(a, b);
                if (n + 1 < NP) {
                    a -= __uint_as_float(w[n][i] << 16);
                    b -= __uint_as_float(w[n][i] & 0xffff0000u);
                }
            }
        }
    }
#pragma unroll
    for (int n = 0; n < NP; ++n) {
        const u32x4 v = {w[n][0], w[n][1], w[n][2], w[n][3]};
        out[n] = __builtin_bit_cast(typename Half16<V>::v8, v);
    }
}

template <int NB, int BITS, typename T, int QT> struct WaveState {
    static constexpr int DV = RawTile<NB, BITS>::DV;
    float m[QT], l[QT];                       // of the lane's column: running maximum of the scores (unscaled), this lane's part of the sum
    f32x4 acc[QT][DV];                        // out^T: rows 4g + i of operand j are numbers DV (4g + i) + j of the column
    __device__ __forceinline__ void reset() {
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            m[t] = -INFINITY;
            l[t] = 0.f;
#pragma unroll
            for (int j = 0; j < DV; ++j) acc[t][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
        }
    }
};

// scores of 32 keys: element i of s[t] belongs to key v_row(g, i) and the lane's column t
template <int NB, int BITS, typename T, int QT>
__device__ __forceinline__ void tile_scores(const RawTile<NB, BITS>& r, const bf16x8 (&qf)[QT][AttnTerms<T>::q][NB], f32x4 (&s)[QT][2], int lane) {
    constexpr int NQ = AttnTerms<T>::q;
    const int g = lane >> 4;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int t = 0; t < QT; ++t) s[t][h] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < NB; ++j) {                             // unit NB g + j of 8 numbers lies in block (NB g + j) / 4
            const bf16x8 kf = decode8<BITS>(&r.k[h][j * BITS / 4], scale_of(r.ks[h], NB == 1 ? 0 : NB == 2 ? g >> 1 : NB == 4 ? g : (3 * g + j) >> 2));
#pragma unroll
            for (int t = 0; t < QT; ++t)
#pragma unroll
                for (int n = NQ - 1; n >= 0; --n) s[t][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[t][n][j], s[t][h], 0, 0, 0);
        }
    }
}

// scores of NS x 32 keys -> weights, as operands of the second product; the state follows the new maximum
template <int NB, int BITS, typename T, int QT, int NS, bool HALF = false>
__device__ __forceinline__ void tile_weights(const f32x4 (&s)[QT][2 * NS], WaveState<NB, BITS, T, QT>& st,
                                             typename Half16<typename Products<T, HALF>::value>::v8 (&pf)[NS][QT][Products<T, HALF>::p], f32x4 (&lsum)[QT], int k0, bool masked, const int (&lo)[QT], const int (&hi)[QT], float c, int lane) {
    constexpr int DV = RawTile<NB, BITS>::DV;
    const int g = lane >> 4;
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        float x[NS][8];
#pragma unroll
        for (int u = 0; u < NS; ++u)
#pragma unroll
            for (int i = 0; i < 8; ++i) x[u][i] = s[t][2 * u + (i >> 2)][i & 3];
        if (masked) {
#pragma unroll
            for (int u = 0; u < NS; ++u)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int key = k0 + 32 * u + v_row(g, i);
                    x[u][i] = (key <= hi[t] && key >= lo[t]) ? x[u][i] : -INFINITY;
                }
        }
        // (by v_med3 with a number above every score: fmaxf would quiet each score in an instruction of its own first)
        float top[4 * NS];
#pragma unroll
        for (int k = 0; k < 4 * NS; ++k) top[k] = __builtin_amdgcn_fmed3f(x[k >> 2][2 * (k & 3)], x[k >> 2][2 * (k & 3) + 1], 3.0e38f);
#pragma unroll
        for (int k = 2 * NS; k > 0; k >>= 1)
#pragma unroll
            for (int i = 0; i < k; ++i) top[i] = __builtin_amdgcn_fmed3f(top[i], top[i + k], 3.0e38f);
        // The state moves to a new reference only when a score passes the old one by more than 2^growth (weights then stay below
        // 2^(growth + lift): no precision is lost, the operands have the range): with the running maximum itself some column of 16 moves in most
        // tiles, and every move costs a multiplication per accumulator.  The lanes of a column hold the same reference, so each asks
        // for its own scores only.
        if (__any(__builtin_fmaf(top[0], c, -st.m[t] * c) > Products<T, HALF>::growth || st.m[t] == -INFINITY)) {
            const float mx = rows_max(top[0]);
            const float mn = fmaxf(st.m[t], mx);
            const float corr = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((st.m[t] - mn) * c);
            st.m[t] = mn;
            if constexpr (kSumByProduct<T, HALF>) lsum[t] *= corr;
            else st.l[t] *= corr;
#pragma unroll
            for (int j = 0; j < DV; ++j) st.acc[t][j] *= corr;
        }
        const float mc = (st.m[t] == -INFINITY ? 0.f : st.m[t] * c) - Products<T, HALF>::lift;
#pragma unroll
        for (int u = 0; u < NS; ++u) {
            float p[8];
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[u][i], c, -mc));
                sum += p[i];
            }
            if constexpr (!kSumByProduct<T, HALF>) st.l[t] += sum;
            split_p<Products<T, HALF>::p, typename Products<T, HALF>::value>(p, pf[u][t]);
        }
    }
}

// acc += V^T P^T, two operands (the even and the odd numbers of a pair) at a time
template <int NB, int BITS, typename T, int QT>
__device__ __forceinline__ void tile_values(const RawTile<NB, BITS>& r, WaveState<NB, BITS, T, QT>& st, const bf16x8 (&pf)[QT][AttnTerms<T>::p], int lane) {
    constexpr int NP = AttnTerms<T>::p, DV = RawTile<NB, BITS>::DV;
    const int li = lane & 15;
    float sc[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) sc[i] = scale_of(r.vs[i], NB == 1 ? 0 : NB == 2 ? li >> 3 : li >> 2);
#pragma unroll
    for (int j = 0; j < DV / 2; ++j) {
        u32x4 vf[2];
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const unsigned a = decode_pair<BITS>(r.v[i], j, sc[i]), b = decode_pair<BITS>(r.v[i + 1], j, sc[i + 1]);
            vf[0][i >> 1] = __builtin_amdgcn_perm(b, a, 0x05040100u);
            vf[1][i >> 1] = __builtin_amdgcn_perm(b, a, 0x07060302u);
        }
#pragma unroll
        for (int n = NP - 1; n >= 0; --n)
#pragma unroll
            for (int t = 0; t < QT; ++t)
#pragma unroll
                for (int o = 0; o < 2; ++o)
                    st.acc[t][2 * j + o] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, vf[o]), pf[t][n], st.acc[t][2 * j + o], 0, 0, 0);
    }
}

// value rows whose block is not finite, and rows before `beg`, which nobody sees: zeros in their place, and NaN as the mark of the columns
// that see one
template <int NB, int BITS, typename T, int QT>
__device__ __forceinline__ void clean_values(RawTile<NB, BITS>& r, float (&mark)[QT], int k0, int beg, const int (&lo)[QT], const int (&hi)[QT], int lane) {
    constexpr int VW = RawTile<NB, BITS>::VW;
    const int li = lane & 15, g = lane >> 4;
    const int acc_block = NB == 1 ? 0 : NB == 2 ? g >> 1 : g, own_block = NB == 1 ? 0 : NB == 2 ? li >> 3 : li >> 2;
    unsigned part = 0;                                             // byte b, bit i: row v_row(g, i) is not finite in block b
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int b = 0; b < NB; ++b) part |= (((r.vs[i] >> (8 * b)) & 255u) >= 228u ? 1u : 0u) << (8 * b + i);
    unsigned rows = 0;                                             // bit k: key k0 + k is not finite in the block of this lane's accumulators
#pragma unroll
    for (int gg = 0; gg < 4; ++gg) {
        const unsigned m = (unsigned)__builtin_amdgcn_readlane((int)part, 16 * gg) >> (8 * acc_block) & 255u;
        rows |= (m & 15u) << (4 * gg) | (m >> 4) << (16 + 4 * gg);
    }
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        const int first = max(lo[t] - k0, 0), last = min(hi[t] - k0, 31);
        const unsigned seen = first <= last ? (~0u >> (31 - last)) & (~0u << first) : 0u;
        if (rows & seen) mark[t] = __builtin_nanf("");
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (((r.vs[i] >> (8 * own_block)) & 255u) >= 228u || k0 + v_row(g, i) < beg) {
            r.vs[i] = 0;
#pragma unroll
            for (int w = 0; w < VW; ++w) r.v[i][w] = 0;
        }
}

// the fresh row (codes of key and value, then their scale words) in place of what the cache still holds at its position
template <int NB, int BITS>
__device__ __forceinline__ void take_fresh_key(RawTile<NB, BITS>& r, const unsigned char* fresh, int k0, int pos, int lane) {
    constexpr int RB = 4 * NB * BITS, KB = RB / 4, KW = RawTile<NB, BITS>::KW;
    const int li = lane & 15, g = lane >> 4;
    unsigned kw[KW];                                               // (read by all lanes, then selected: a read under the condition is a branch a word)
    lds_words<KB>(fresh + g * KB, kw);
    const unsigned ks = *(const unsigned*)(fresh + 2 * RB);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const bool here = k0 + li + 16 * h == pos;
#pragma unroll
        for (int i = 0; i < KW; ++i) r.k[h][i] = here ? kw[i] : r.k[h][i];
        r.ks[h] = here ? ks : r.ks[h];
    }
}
template <int NB, int BITS>
__device__ __forceinline__ void take_fresh_value(RawTile<NB, BITS>& r, const unsigned char* fresh, int k0, int pos, int lane) {
    constexpr int RB = 4 * NB * BITS, DV = RawTile<NB, BITS>::DV, VB = DV * BITS / 8, VW = RawTile<NB, BITS>::VW;
    const int li = lane & 15, g = lane >> 4;
    unsigned vw[VW];
    lds_words<VB>(fresh + RB + (NB == 3 ? min(li, 11) : li) * VB, vw);
    const unsigned vs = *(const unsigned*)(fresh + 2 * RB + 4);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const bool here = k0 + v_row(g, i) == pos;
#pragma unroll
        for (int w = 0; w < VW; ++w) r.v[i][w] = here ? vw[w] : r.v[i][w];
        r.vs[i] = here ? vs : r.vs[i];
    }
}

// the columns of a lane: positions that each sees
template <int QT> __device__ __forceinline__ void lane_columns(const AttnCacheArgs& a, const KvRow& r, int c0, int li, int (&col)[QT], int (&lo)[QT], int (&hi)[QT]) {
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        col[t] = c0 + 16 * t + li;
        const int step = col[t] / a.G;
        const int qp = a.causal ? r.pos + step : r.pos + r.cnt - 1;
        hi[t] = (col[t] < a.N && step < r.cnt && r.e >= 0) ? min(min(qp, a.g.S - 1), a.max_len - 1) : -1;
        lo[t] = a.window ? max(qp - a.window + 1, 0) : 0;
    }
}

// query operands: numbers 8 NB g + 8 j .. + 7 of the lane's column, as a sum of bf16 terms (cut, not rounded: the rest is exact)
template <int NB, typename T, int QT, bool HALF = false>
__device__ __forceinline__ void load_queries(const AttnCacheArgs& a, int i, int h, const int (&col)[QT], int g,
                                             typename Half16<typename Products<T, HALF>::key>::v8 (&qf)[QT][Products<T, HALF>::q][NB]) {
    typedef typename Products<T, HALF>::key K;
    constexpr int NQ = Products<T, HALF>::q;
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        const int step = col[t] / a.G, hq = h * a.G + col[t] - step * a.G;
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            if (col[t] < a.N) kv_load8<T>((const T*)a.q.p + (long)i * a.q.row + (long)step * a.q.step + (long)hq * a.q.head + 8 * (NB * g + j), a.q_vec, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float rest = x[e];
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
                    const float cut = NQ > 1 ? __uint_as_float(__float_as_uint(rest) & 0xffff0000u) : rest;
                    qf[t][n][j][e] = (K)cut;
                    rest -= cut;
                }
            }
        }
    }
}

// a lane's columns: numbers 4 DV g .. + 4 DV - 1, to the output (one split) or, not yet divided, to the scratch
template <int NB, int BITS, typename T, int QT>
__device__ __forceinline__ void store_columns(const AttnCacheArgs& a, const WaveState<NB, BITS, T, QT>& st, int u, int i, int h, int sp, const int (&col)[QT],
                                              const int (&lo)[QT], const int (&hi)[QT], int g) {
    constexpr int D = 32 * NB, DV = RawTile<NB, BITS>::DV;
    if (NB == 3 && g == 3) return;
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        if (col[t] >= a.N) continue;
        if (a.nsplit > 1) {
            float* y = a.part + (((long)sp * a.g.n * a.g.H + u) * a.N + col[t]) * (D + 2);
#pragma unroll
            for (int d = 0; d < 4 * DV; d += 2) *(f32x2*)(y + 4 * DV * g + d) = (f32x2){st.acc[t][d % DV][d / DV], st.acc[t][(d + 1) % DV][(d + 1) / DV]};
            if (g == 0) *(f32x2*)(y + D) = (f32x2){st.m[t], st.l[t]};
            continue;
        }
        const int step = col[t] / a.G, hq = h * a.G + col[t] - step * a.G;
        const bool none = lo[t] > hi[t];
        const float inv = 1.0f / st.l[t];
        T* o = (T*)a.out.p + (long)i * a.out.row + (long)step * a.out.step + (long)hq * a.out.head + 4 * DV * g;
#pragma unroll
        for (int q = 0; q < DV / 2; ++q) {                         // 8 consecutive numbers at a time
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) { const int d = 8 * q + e; y[e] = none ? 0.f : st.acc[t][d % DV][d / DV] * inv; }
            if constexpr (sizeof(T) == 4) {
                *(f32x4*)(o + 8 * q) = (f32x4){y[0], y[1], y[2], y[3]};
                *(f32x4*)(o + 8 * q + 4) = (f32x4){y[4], y[5], y[6], y[7]};
            } else {
                typename Half16<T>::v8 v;
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = kv_result<T>(y[e]);
                *(typename Half16<T>::v8*)(o + 8 * q) = v;
            }
        }
    }
}

// The step's own key and value (args.kn, args.vn): codes to the cache (`stores`: one wave of the item) and to this wave's LDS
// row `fr` -- codes of the key, of the value, then their scale words -- for the tile that holds its position.  Returns that
// position if it lies in [start, stop), -1 otherwise.
template <int NB, int BITS, typename T>
__device__ __forceinline__ int append_row(const AttnCacheArgs& a, const KvRow& r, int i, int h, int sp, int start, int stop, int end, bool stores,
                                          unsigned char* fr, int lane) {
    constexpr int RB = 4 * NB * BITS;
    // (a position that max_len hides is stored all the same, by the first split)
    const bool sees = r.pos >= start && r.pos < stop;
    if (!a.kn.p || r.e < 0 || !(sees || (sp == 0 && r.pos >= end && r.pos < a.g.S))) return -1;
    const int p = lane & 15, kv = lane >> 4;                       // lanes 0 .. 15: the key row, 16 .. 31: the value row, 8 numbers each
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    const bool on = lane < 32 && p < 4 * NB;
    const KvOperand<const void>& o = kv ? a.vn : a.kn;
    if (on) kv_load8<T>((const T*)o.p + (long)i * o.row + (long)h * o.head + 8 * p, a.new_vec, x);
    int from = i;                                                  // an episode listed twice: the last listing is the one that is stored and seen
    if (a.g.idx) {
        int last = i;
        for (int j0 = i + 1; j0 < a.g.n; j0 += 512) {              // eight loads in flight
            int other[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) other[q] = a.g.idx[min(j0 + 64 * q + lane, a.g.n - 1)];
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const int j = j0 + 64 * q + lane;
                last = j < a.g.n && other[q] == r.e ? j : last;
            }
        }
        if (__any(last != i)) {
#pragma unroll
            for (int q = 32; q > 0; q >>= 1) last = max(last, __shfl_xor(last, q, 64));
            from = __builtin_amdgcn_readfirstlane(last);
            if (on) kv_load8<T>((const T*)o.p + (long)from * o.row + (long)h * o.head + 8 * p, a.new_vec, x);
        }
    }
    const unsigned sb = kv_scale_byte<BITS>(kv_block_top(x));
    unsigned cw[BITS / 4];
    kv_encode8<BITS>(x, sb, cw);
    if (lane < 2) *(unsigned*)(fr + 2 * RB + 4 * lane) = 0u;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (on) {
#pragma unroll
        for (int q = 0; q < BITS / 4; ++q) *(unsigned*)(fr + kv * RB + p * BITS + 4 * q) = cw[q];
        if ((p & 3) == 0) fr[2 * RB + 4 * kv + (p >> 2)] = (unsigned char)sb;
        if (from == i && stores) {
            unsigned char* cc = a.g.codes + kv * a.g.ckv + (long)r.e * a.g.ce + (long)h * a.g.ch + (long)r.pos * RB + p * BITS;
            if constexpr (BITS == 4) *(unsigned*)cc = cw[0];
            else *(uint2*)cc = make_uint2(cw[0], cw[BITS / 4 - 1]);
            if ((p & 3) == 0) a.g.scales[kv * a.g.skv + (long)r.e * a.g.se + (long)h * a.g.sh + (long)r.pos * 4 + (p >> 2)] = (unsigned char)sb;
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    return sees ? r.pos : -1;
}

// Items: (split, row, key head, column group).  A workgroup of four waves takes one item with the keys dealt out in tiles
// (kw = 4), or four items: neighbouring column groups of one (row, head), which read the same rows, or, with one column
// group, four (row, head) pairs.  (row, head) runs fastest over the workgroups, so that the column groups of one pair meet in
// one XCD's L2; the last column groups, which see the most keys under a causal mask, start first.
// Memory-bound where it matters, one position over long histories: 48 rows x 32 / 8 heads of 128 over 7001 to 16383 positions in 4 bits
// read 610 MB in 126 us (4.8 TB/s, the rate of a large copy), 160 x 16 / 4 heads of 64 over the last 1000 in 8 bits 85 MB in 20 us.
// Short windows (64 x 8 heads x 32 steps of 96, fp32: 9 us) are one tile a wave: the latency of its dependent loads.
// Registers spilled under the launch bounds: fp16 heads of 128, 2 (4 bits) and 13 (8 bits) with 16 columns, 14 (8 bits) with 32; fp32 heads of 96, 2
// and 10; none elsewhere.
template <int NB, int BITS, typename T, int QT>
__global__ __launch_bounds__(256, narrow_groups(KvElem<T>::code, NB, QT)) void attn_cache_kernel(AttnCacheArgs a) {
    constexpr int D = 32 * NB, RB = 4 * NB * BITS, DV = RawTile<NB, BITS>::DV, NQ = AttnTerms<T>::q;
    constexpr int MROW = D + 4;                                    // padded row of the merge buffer
    __shared__ __attribute__((aligned(16))) unsigned char fresh_rows[4][2 * RB + 16];
    __shared__ __attribute__((aligned(16))) float merge[4 * 16 * MROW];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int li = lane & 15, g = lane >> 4;
    const int U = a.g.n * a.g.H;
    int u, cg, sp = 0;
    {
        int b = blockIdx.x;
        if (a.kw == 4) {
            u = b % U;
            b /= U;
            cg = a.CG - 1 - b % a.CG;
            sp = b / a.CG;
        } else if (a.CG == 1) {
            u = b * 4 + w;
            cg = 0;
        } else {
            u = b % U;
            cg = ((a.CG + 3) / 4 - 1 - b / U) * 4 + w;
        }
    }
    if (u >= U || cg >= a.CG) return;                              // (only with kw = 1: no barrier follows)
    const int i = u / a.g.H, h = u - i * a.g.H;
    const KvRow r = kv_row(a.g, i);
    const int c0 = cg * 16 * QT, c1 = min(c0 + 16 * QT, a.N) - 1;
    const KeyRange kr = key_range(a, r, c0, c1);
    const int start = (kr.beg & ~31) + sp * a.chunk, stop = min(kr.end, start + a.chunk);
    if (sp > 0 && start >= stop) return;                           // the whole workgroup: the item has fewer splits
    const bool whole = a.nsplit == 1;

    int lo[QT], hi[QT], col[QT];
    lane_columns<QT>(a, r, c0, li, col, lo, hi);

    TileSource src;
    {
        const long e = max(r.e, 0);
        src.k = a.g.codes + e * a.g.ce + (long)h * a.g.ch;
        src.v = src.k + a.g.ckv;
        src.ks = a.g.scales + e * a.g.se + (long)h * a.g.sh;
        src.vs = src.ks + a.g.skv;
    }
    WaveState<NB, BITS, T, QT> st;
    const int first = start + (a.kw == 4 ? 32 * w : 0), stride = a.kw * 32;
    // one tile's registers: the next keys are requested once the scores stand, the next values once the second product has read its own
    RawTile<NB, BITS> raw;
    if (first < stop) {                                            // on their way while the fresh row and the queries are dealt with
        load_keys<NB, BITS>(raw, src, first, stop - first, lane);
        load_values<NB, BITS>(raw, src, first, stop - first, lane);
    }
    unsigned char* fr = fresh_rows[w];
    const int fresh_pos = append_row<NB, BITS, T>(a, r, i, h, sp, start, stop, kr.end, cg == 0 && (a.kw == 1 || w == 0), fr, lane);
    bf16x8 qf[QT][NQ][NB];
    load_queries<NB, T, QT>(a, i, h, col, g, qf);
    auto keys = [&](int k0) {
        load_keys<NB, BITS>(raw, src, k0, stop - k0, lane);
        if (fresh_pos >= k0 && fresh_pos < k0 + 32) take_fresh_key<NB, BITS>(raw, fr, k0, fresh_pos, lane);
    };
    auto values = [&](int k0) {
        load_values<NB, BITS>(raw, src, k0, stop - k0, lane);
        if (fresh_pos >= k0 && fresh_pos < k0 + 32) take_fresh_value<NB, BITS>(raw, fr, k0, fresh_pos, lane);
    };
    st.reset();
    float mark[QT] = {};
    if (fresh_pos >= first && fresh_pos < first + 32) {
        take_fresh_key<NB, BITS>(raw, fr, first, fresh_pos, lane);
        take_fresh_value<NB, BITS>(raw, fr, first, fresh_pos, lane);
    }
    for (int k0 = first; k0 < stop; k0 += stride) {
        const bool more = k0 + stride < stop;
        const bool masked = k0 + 31 > kr.hi_all || k0 + 31 >= stop || k0 < kr.lo_all;
        f32x4 s[QT][2];
        bf16x8 pf[1][QT][AttnTerms<T>::p];
        tile_scores<NB, BITS, T, QT>(raw, qf, s, lane);
        if (more) keys(k0 + stride);
        f32x4 unread[QT];                                            // (the sums of products are the wide form's)
        tile_weights<NB, BITS, T, QT, 1>(s, st, pf, unread, k0, masked, lo, hi, a.c, lane);
        unsigned suspect = 0;
        if (masked) {
#pragma unroll
            for (int i = 0; i < 8; ++i) suspect |= raw.vs[i] & (raw.vs[i] << 1) & (raw.vs[i] << 2) & 0x80808080u;
        }
        if (__any(suspect != 0) || k0 < kr.beg) clean_values<NB, BITS, T, QT>(raw, mark, k0, kr.beg, lo, hi, lane);
        tile_values<NB, BITS, T, QT>(raw, st, pf[0], lane);
        if (more) values(k0 + stride);
    }
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        st.l[t] = rows_sum(st.l[t]);
#pragma unroll
        for (int j = 0; j < DV; ++j) st.acc[t][j] += mark[t];
    }

    const long part_row = ((long)sp * U + u) * a.N;
    if (a.kw == 1) {
        store_columns<NB, BITS, T, QT>(a, st, u, i, h, sp, col, lo, hi, g);
        return;
    }
    // four waves saw different keys of the same columns: merge through LDS, 16 columns at a time
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        if (c0 + 16 * t >= a.N) break;                             // uniform
        if (t > 0) __syncthreads();
        float* mine = merge + (w * 16 + li) * MROW;
        if (!(NB == 3 && g == 3)) {
#pragma unroll
            for (int d = 0; d < 4 * DV; d += 4)
                *(f32x4*)(mine + 4 * DV * g + d) = (f32x4){st.acc[t][d % DV][d / DV], st.acc[t][(d + 1) % DV][(d + 1) / DV],
                                                           st.acc[t][(d + 2) % DV][(d + 2) / DV], st.acc[t][(d + 3) % DV][(d + 3) / DV]};
        }
        if (g == 0) { mine[D] = st.m[t]; mine[D + 1] = st.l[t]; }
        __syncthreads();
        for (int q = threadIdx.x; q < 16 * (D / 4); q += 256) {
            const int c = q / (D / 4), d = (q % (D / 4)) * 4, cc = c0 + 16 * t + c;
            if (cc >= a.N) continue;
            float m = -INFINITY, l = 0.f;
            f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < 4; ++k) m = fmaxf(m, merge[(k * 16 + c) * MROW + D]);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float* from = merge + (k * 16 + c) * MROW;
                const float f = from[D] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((from[D] - m) * a.c);
                l += from[D + 1] * f;
                o += *(const f32x4*)(from + d) * f;
            }
            const int step = cc / a.G, hq = h * a.G + cc - step * a.G;
            if (whole) {
                const int qp = a.causal ? r.pos + step : r.pos + r.cnt - 1;
                const int last = min(min(qp, a.g.S - 1), a.max_len - 1), beg = a.window ? max(qp - a.window + 1, 0) : 0;
                const bool none = r.e < 0 || step >= r.cnt || beg > last;
                const float inv = 1.0f / l;
                T* y = (T*)a.out.p + (long)i * a.out.row + (long)step * a.out.step + (long)hq * a.out.head + d;
                if constexpr (sizeof(T) == 4) {
                    *(f32x4*)y = none ? (f32x4){0.f, 0.f, 0.f, 0.f} : o * inv;
                } else {
                    typename Half16<T>::v4 v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = kv_result<T>(none ? 0.f : o[e] * inv);
                    *(typename Half16<T>::v4*)y = v;
                }
            } else {
                float* y = a.part + (part_row + cc) * (D + 2);
                *(f32x2*)(y + d) = (f32x2){o[0], o[1]};
                *(f32x2*)(y + d + 2) = (f32x2){o[2], o[3]};
                if (d == 0) *(f32x2*)(y + D) = (f32x2){m, l};
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------
// Many columns a row (whole windows, chunks): a workgroup's four waves own neighbouring column groups of one (row, head) and walk
// over its keys together.  Converting a tile takes as many vector instructions as a column group's softmax, so the four waves
// convert 64 keys once between them -- a wave its 16 keys and half the numbers of its 32 value rows -- into LDS, in the order in
// which the matrix operands are read (16 bytes a lane, no conflicts), while the previous tile is being multiplied: two buffers,
// one barrier a tile.
// A tile of 64 keys x 32 columns x 64 numbers is 36 products (576 cycles) and 190 vector instructions a wave in bf16, 32 of them
// exponentials.  8 windows of 2047 steps, 12 heads of 64, 4 bits: bf16 100 to 106 us by the machine (512 TFLOP/s at 100, counting only visible
// keys), fp16 131, fp32 174; 8 x 500 steps after 2500 to 7600 positions, 32 / 8 heads of 128, bf16 395 us.  With a kernel of the narrow
// form the two took 158 and 767 us.  Bound by vector issue and waiting: of a SIMD's cycles 21 % are products and 41 % the issue of vector
// instructions (the exponentials take longer than counted there) in the first, 35 and 32 % in the second, and the waves wait a third.
// Products do not exclude vector instructions (from another wave about half of an exponential, maximum and fma mix hides behind them); more waves
// a SIMD do not fit the accumulators, and the fp16 kernels of two column groups for heads of 64 already spill (33 registers in 4 bits, 43 in 8:
// the bf16 walk that they contain needs two query terms).
template <int NB, int BITS> struct WideTile {
    static constexpr int DV = RawTile<NB, BITS>::DV, KW = RawTile<NB, BITS>::KW;
    static constexpr int PW = DV / 4 > 0 ? DV / 4 : 1;             // pairs of numbers of a value row that one wave converts
    static constexpr int PB = PW * BITS / 4;                       // bytes of those
    static constexpr int frags = 4 * NB + 2 * DV;                  // operands of 64 lanes x 16 bytes: 4 x 16 keys, then 2 x 32 value rows
    static constexpr int bytes = frags * 1024 + 64;                // and a row mask per (32 keys, block) of the value rows that are not finite
    unsigned k[KW], v[8][1], ks, vs[8];
    unsigned own;                                                  // value scale word of the key that ks belongs to (range check of the fp16 operands)
};

template <int NB, int BITS, bool HALF> __device__ __forceinline__ void wide_load(WideTile<NB, BITS>& r, const TileSource& src, int k0, int rows, int lane, int w) {
    constexpr int RB = 4 * NB * BITS, KB = RB / 4, VB = RawTile<NB, BITS>::DV * BITS / 8, PB = WideTile<NB, BITS>::PB;
    const int li = lane & 15, g = lane >> 4;
    const auto kc = rows_of(src.k, k0 + 16 * w, RB, rows - 16 * w), ks = rows_of(src.ks, k0 + 16 * w, 4, rows - 16 * w);
    buffer_words<KB>(kc, li * RB + g * KB, r.k);
    r.ks = __builtin_amdgcn_raw_buffer_load_b32(ks, li * 4, 0, 0);
    if constexpr (HALF) r.own = __builtin_amdgcn_raw_buffer_load_b32(rows_of(src.vs, k0 + 16 * w, 4, rows - 16 * w), li * 4, 0, 0);
    if (NB == 1 && (w & 1)) return;                                // (one pair a lane: two waves do it)
    const int sub = 32 * (w >> 1);
    const auto vc = rows_of(src.v, k0 + sub, RB, rows - sub), vs = rows_of(src.vs, k0 + sub, 4, rows - sub);
    int vl = (NB == 3 ? min(li, 11) : li) * VB + (w & 1) * PB + 4 * g * RB;
    asm("" : "+v"(vl));                                            // (see load_values)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const auto u = __builtin_amdgcn_raw_buffer_load_b128(vs, 16 * g + 64 * h, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) r.vs[4 * h + i] = u[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) buffer_words<PB>(vc, vl + ((i & 3) + 16 * (i >> 2)) * RB, r.v[i]);
}

// `edge`: the tile has keys that some column does not see: blocks that are not finite are taken out and named in the masks; so are
// the tile's first `before` rows, which no column sees
// `least`, `most`: over the scale bytes of the tile's keys (a wave looks at its 16), as the top bits of a word, `least` less 1: the
// zeros of rows that do not exist wrap around and pass
template <int NB, int BITS, typename T, bool HALF>
__device__ __forceinline__ void wide_convert(WideTile<NB, BITS>& r, unsigned char* buf, bool edge, int before, unsigned& least, unsigned& most, int lane, int w) {
    typedef WideTile<NB, BITS> W;
    typedef typename Products<T, HALF>::key K;
    typedef typename Products<T, HALF>::value V;
    constexpr int key_up = KvElem<K>::code == DT_F16 ? kUp<BITS> : 0, value_up = HALF ? kUp<BITS> : 0;
    const int li = lane & 15, g = lane >> 4;
    auto meet = [&](unsigned word, unsigned passes) {              // blocks whose byte is `passes` or more have no say
#pragma unroll
        for (int b = 0; b < NB; ++b) {                             // (what lies below the byte decides nothing)
            const unsigned y = word << (24 - 8 * b);
            const bool pass = passes < 256u && y >= passes << 24;
            least = min(least, pass ? ~0u : y - (1u << 24));
            most = max(most, pass ? 0u : y);
        }
    };
    if constexpr (HALF) {
        const bool unseen = edge && 16 * w + li < before;          // (what nobody sees decides nothing; an edge's rows that are not finite are taken out)
        if constexpr (KvElem<K>::code == DT_F16) meet(unseen ? 0u : r.ks, 255u);       // (a key that is no number is none in either type)
        if (edge) meet(unseen ? 0u : r.own, 228u);
        else meet(r.own, 256u);
    }
#pragma unroll
    for (int j = 0; j < NB; ++j)
        *(typename Half16<K>::v8*)(buf + (w * NB + j) * 1024 + lane * 16) =
            decode8<BITS, K>(&r.k[j * BITS / 4], scale_up<key_up>(r.ks, NB == 1 ? 0 : NB == 2 ? g >> 1 : NB == 4 ? g : (3 * g + j) >> 2));
    if (NB == 1 && (w & 1)) return;
    const int block = NB == 1 ? 0 : NB == 2 ? li >> 3 : NB == 3 ? min(li, 11) >> 2 : li >> 2;
    if (edge) {
        unsigned part = 0;                                         // byte b, bit i: row v_row(g, i) is not finite in block b
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int b = 0; b < NB; ++b) part |= (((r.vs[i] >> (8 * b)) & 255u) >= 228u ? 1u : 0u) << (8 * b + i);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (((r.vs[i] >> (8 * block)) & 255u) >= 228u || 32 * (w >> 1) + v_row(g, i) < before) r.vs[i] = r.v[i][0] = 0;
        unsigned rows[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            rows[b] = 0;
#pragma unroll
            for (int gg = 0; gg < 4; ++gg) {
                const unsigned m = (unsigned)__builtin_amdgcn_readlane((int)part, 16 * gg) >> (8 * b) & 255u;
                rows[b] |= (m & 15u) << (4 * gg) | (m >> 4) << (16 + 4 * gg);
            }
        }
        if ((w & 1) == 0 && lane == 0) *(u32x4*)(buf + W::frags * 1024 + 16 * (w >> 1)) = (u32x4){rows[0], rows[1], rows[2], rows[3]};
    }
    float sc[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) sc[i] = scale_up<value_up>(r.vs[i], block);
    unsigned char* to = buf + (4 * NB + (w >> 1) * W::DV + (w & 1) * 2 * W::PW) * 1024 + lane * 16;
#pragma unroll
    for (int j = 0; j < W::PW; ++j) {
        u32x4 vf[2];
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const unsigned a = decode_pair<BITS, V>(r.v[i], j, sc[i]), b = decode_pair<BITS, V>(r.v[i + 1], j, sc[i + 1]);
            vf[0][i >> 1] = __builtin_amdgcn_perm(b, a, 0x05040100u);
            vf[1][i >> 1] = __builtin_amdgcn_perm(b, a, 0x07060302u);
        }
        *(u32x4*)(to + 2 * j * 1024) = vf[0];
        *(u32x4*)(to + (2 * j + 1) * 1024) = vf[1];
    }
}

// whether a block of rows beg .. stop - 1 whose scale byte is below LO holds a number other than zero.  Read again only after a walk that met
// such bytes: 8 windows of 2047 steps, 12 heads of 64, with zeros in every 50th row take 110 us (bf16, 4 bits) and 141 (fp16, 8 bits), without
// any 105 and 119; a second walk costs 100 and more.
template <int NB, int BITS, int LO>
__device__ __forceinline__ bool low_numbers(const unsigned char* rows, const unsigned char* scales, int start, int stop, int beg, int lane, int w) {
    constexpr int RB = 4 * NB * BITS, KB = RB / 4;
    constexpr unsigned magnitude = BITS == 4 ? 0x77777777u : 0x7f7f7f7fu;
    asm volatile("" : "+v"(lane), "+s"(start), "+s"(stop));        // (nothing of this is worth a register of the walk before it)
    const int li = lane & 15, g = lane >> 4;
    bool found = false;
    for (int k0 = start + 16 * w; k0 < stop; k0 += 64) {           // a wave takes 16 rows, a lane a quarter of one
        unsigned c[RawTile<NB, BITS>::KW];
        buffer_words<KB>(rows_of(rows, k0, RB, stop - k0), li * RB + g * KB, c);
        const unsigned word = __builtin_amdgcn_raw_buffer_load_b32(rows_of(scales, k0, 4, stop - k0), li * 4, 0, 0);
#pragma unroll
        for (int j = 0; j < NB; ++j) {                             // (units of 8 numbers, as in tile_scores)
            const int block = NB == 1 ? 0 : NB == 2 ? g >> 1 : NB == 4 ? g : (3 * g + j) >> 2;
            const unsigned some = (c[j * BITS / 4] | c[j * BITS / 4 + BITS / 4 - 1]) & magnitude;
            found |= some != 0u && (word >> (8 * block) & 255u) < LO && k0 + li >= beg;
        }
    }
    return found;
}

// a workgroup's walk over its keys; true: a block does not fit the fp16 operands, the state is void (the same for all threads)
template <int NB, int BITS, typename T, int QT, bool HALF>
__device__ __forceinline__ bool wide_walk(const AttnCacheArgs& a, const TileSource& src, const KeyRange& kr, const KeyRange& own, int start, int stop, int i, int h,
                                          const int (&col)[QT], const int (&lo)[QT], const int (&hi)[QT], WaveState<NB, BITS, T, QT>& st, unsigned char* lds,
                                          int lane, int w) {
    typedef Products<T, HALF> P;
    typedef Half16<typename P::key> HK;
    typedef Half16<typename P::value> HV;
    typedef WideTile<NB, BITS> W;
    constexpr int DV = RawTile<NB, BITS>::DV, NQ = P::q, NP = P::p;
    const int g = lane >> 4;
    typename HK::v8 qf[QT][NQ][NB];
    load_queries<NB, T, QT, HALF>(a, i, h, col, g, qf);
    st.reset();
    float mark[QT] = {};
    constexpr float key_down = KvElem<typename P::key>::code == DT_F16 ? 1.f / (1 << kUp<BITS>) : 1.f;      // scores come out 2^kUp times as large
    f32x4 lsum[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t) lsum[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
    typename HV::v8 ones;
#pragma unroll
    for (int e = 0; e < 8; ++e) ones[e] = (typename P::value)1.f;
    unsigned least = ~0u;
    unsigned most = 0;
    auto edge = [&](int k0) { return k0 + 63 > kr.hi_all || k0 + 64 > stop || k0 < kr.lo_all; };
    WideTile<NB, BITS> raw;
    if (start < stop) {
        wide_load<NB, BITS, HALF>(raw, src, start, stop - start, lane, w);
        wide_convert<NB, BITS, T, HALF>(raw, lds, edge(start), kr.beg - start, least, most, lane, w);
        if (start + 64 < stop) wide_load<NB, BITS, HALF>(raw, src, start + 64, stop - start - 64, lane, w);
    }
    __syncthreads();
    int at = 0;
    for (int k0 = start; k0 < stop; k0 += 64, at ^= 1) {
        const unsigned char* buf = lds + at * W::bytes;
        const bool work = k0 < own.end && k0 + 64 > own.beg;       // somebody in this wave sees a key of the tile
        const bool more = k0 + 64 < stop;
        typename HV::v8 pf[2][QT][NP];
        if (work) {
            f32x4 s[QT][4];
#pragma unroll
            for (int hh = 0; hh < 4; ++hh)
#pragma unroll
                for (int t = 0; t < QT; ++t) s[t][hh] = (f32x4){0.f, 0.f, 0.f, 0.f};
            // (neighbouring products go to different accumulators: one that waits for its predecessor stalls the matrix pipe)
#pragma unroll
            for (int n = NQ - 1; n >= 0; --n)
#pragma unroll
                for (int j = 0; j < NB; ++j)
#pragma unroll
                    for (int hh = 0; hh < 4; ++hh) {
                        const typename HK::v8 kf = *(const typename HK::v8*)(buf + (hh * NB + j) * 1024 + lane * 16);
#pragma unroll
                        for (int t = 0; t < QT; ++t) s[t][hh] = HK::mfma32(kf, qf[t][n][j], s[t][hh]);
                    }
            const bool masked = k0 + 63 > own.hi_all || k0 + 64 > stop || k0 < own.lo_all;
            tile_weights<NB, BITS, T, QT, 2, HALF>(s, st, pf, lsum, k0, masked, lo, hi, a.c * key_down, lane);
        }
        if (more) {                                                // the next tile into the other buffer, the one behind it on its way
            wide_convert<NB, BITS, T, HALF>(raw, lds + (at ^ 1) * W::bytes, edge(k0 + 64), kr.beg - k0 - 64, least, most, lane, w);
            if (k0 + 128 < stop) wide_load<NB, BITS, HALF>(raw, src, k0 + 128, stop - k0 - 128, lane, w);
        }
        if (work) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                if constexpr (kSumByProduct<T, HALF>)
#pragma unroll
                    for (int t = 0; t < QT; ++t) lsum[t] = HV::mfma32(ones, pf[x][t][0], lsum[t]);
#pragma unroll
                for (int j = 0; j < DV; j += 2) {
                    const typename HV::v8 vf[2] = {*(const typename HV::v8*)(buf + (4 * NB + x * DV + j) * 1024 + lane * 16),
                                                   *(const typename HV::v8*)(buf + (4 * NB + x * DV + j + 1) * 1024 + lane * 16)};
#pragma unroll
                    for (int n = NP - 1; n >= 0; --n)
#pragma unroll
                        for (int t = 0; t < QT; ++t)
#pragma unroll
                            for (int o = 0; o < 2; ++o) st.acc[t][j + o] = HV::mfma32(vf[o], pf[x][t][n], st.acc[t][j + o]);
                }
            }
            if (edge(k0)) {
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const unsigned rows = *(const unsigned*)(buf + W::frags * 1024 + 16 * x + 4 * (NB == 1 ? 0 : NB == 2 ? g >> 1 : g));
#pragma unroll
                    for (int t = 0; t < QT; ++t) {
                        const int first = max(lo[t] - k0 - 32 * x, 0), last = min(hi[t] - k0 - 32 * x, 31);
                        const unsigned seen = first <= last ? (~0u >> (31 - last)) & (~0u << first) : 0u;
                        if (rows & seen) mark[t] = __builtin_nanf("");
                    }
                }
            }
        }
        __syncthreads();
    }
    if constexpr (HALF) {
        constexpr int lo_byte = (BITS == 4 ? 127 - 23 : 127 - 15) - kUp<BITS>, hi_byte = (BITS == 4 ? 127 + 13 : 127 + 7) - kUp<BITS>;
        if (__syncthreads_or(most >= (hi_byte + 1u) << 24)) return true;
        if (__builtin_expect(__syncthreads_or(least < (lo_byte - 1u) << 24), 0)) {       // (rare: zeros, or numbers that the operands have lost)
            bool lost = low_numbers<NB, BITS, lo_byte>(src.v, src.vs, start, stop, kr.beg, lane, w);
            if constexpr (KvElem<typename P::key>::code == DT_F16) lost |= low_numbers<NB, BITS, lo_byte>(src.k, src.ks, start, stop, kr.beg, lane, w);
            if (__syncthreads_or(lost)) return true;
        }
    }
    // (exact: splits of one column may be of either kind)
    constexpr float down = HALF ? 1.f / (1 << (int)P::lift) : 1.f, value_down = HALF ? down / (1 << kUp<BITS>) : 1.f;
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        st.m[t] *= key_down;
        st.l[t] = (kSumByProduct<T, HALF> ? lsum[t][0] : rows_sum(st.l[t])) * down;      // (the product's sum is over all keys already)
#pragma unroll
        for (int j = 0; j < DV; ++j) st.acc[t][j] = st.acc[t][j] * value_down + mark[t];
    }
    return false;
}

// The pair (row i, column group cg) that comes at place j when the pairs are in order of how many keys they see, most first.  Histories
// differ by a factor of three in a batch, and a long one that starts last has the chip to itself: 8 chunks of 500 steps after 2500 to
// 7600 positions, 32 / 8 heads of 128: 403 us against
// 540 with the last column groups of all rows first.  Lane = row; a row's groups are
// first .. first + CG - 1 in units of a group's positions, so the place is found by bisection over that unit, a sum over the wave a step.
__device__ __forceinline__ int wave_sum_int(int v) {
    v += __builtin_amdgcn_mov_dpp(v, 0xB1, 0xF, 0xF, true);
    v += __builtin_amdgcn_mov_dpp(v, 0x4E, 0xF, 0xF, true);
    v += __builtin_amdgcn_mov_dpp(v, 0x141, 0xF, 0xF, true);
    v += __builtin_amdgcn_mov_dpp(v, 0x140, 0xF, 0xF, true);
    const auto a = __builtin_amdgcn_permlane32_swap((unsigned)v, (unsigned)v, false, false);
    v = (int)(a[0] + a[1]);
    const auto b = __builtin_amdgcn_permlane16_swap((unsigned)v, (unsigned)v, false, false);
    return __builtin_amdgcn_readfirstlane((int)(b[0] + b[1]));
}
__device__ __forceinline__ KvRow longest_first(const AttnCacheArgs& a, int j, int cols, int lane, int& i, int& cg) {
    KvRow r = kv_row(a.g, min(lane, a.g.n - 1));
    const int groups = lane < a.g.n ? a.CG : 0;
    const int first = r.e >= 0 ? (int)((float)min(max(r.pos, 0), a.max_len) * ((float)a.G / (float)cols)) : 0;
    if (__ballot(first != __builtin_amdgcn_readfirstlane(first)) == 0) {      // whole windows
        const int later = j / a.g.n;
        i = j - later * a.g.n;
        cg = a.CG - 1 - later;
    } else {
        auto above = [&](int t) { return wave_sum_int(min(max(first + a.CG - t, 0), groups)); };      // pairs that see t units or more
        int t = 0, most = (int)((float)a.max_len * ((float)a.G / (float)cols)) + a.CG + 1;            // above(t) > j >= above(most)
        while (most - t > 1) {
            const int mid = t + (most - t) / 2;
            if (above(mid) > j) t = mid;
            else most = mid;
        }
        j -= above(t + 1);
        const bool here = groups && first <= t && t < first + a.CG;
        const unsigned long long rows = __ballot(here);
        const int before = __builtin_amdgcn_mbcnt_hi((unsigned)(rows >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)rows, 0u));
        i = __builtin_ctzll(__ballot(here && before == j));
        cg = t - __builtin_amdgcn_readlane(first, i);
    }
    r.e = __builtin_amdgcn_readlane(r.e, i);
    r.pos = __builtin_amdgcn_readlane(r.pos, i);
    r.cnt = __builtin_amdgcn_readlane(r.cnt, i);
    return r;
}

// Three waves a SIMD where a head is at most 64 numbers (170 registers hold a wave's state then): 8 windows of 2047 steps, 12 heads of
// 64, bf16 123 -> 112 us, fp16 152 -> 136, against two.
template <int NB, int BITS, typename T, int QT>
__global__ __launch_bounds__(256, (NB <= 2 ? 3 : 2)) void attn_cache_wide_kernel(AttnCacheArgs a) {
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int li = lane & 15, g = lane >> 4;
    const int U = a.g.n * a.g.H;
    int i, h, cg, sp = 0;
    KvRow r;
    if (a.longest) {                                               // head fastest
        const int j = blockIdx.x / a.g.H;
        h = blockIdx.x - j * a.g.H;
        r = longest_first(a, j, 64 * QT, lane, i, cg);
    } else {                                                       // (row, head) fastest, then column groups from the last on, then splits
        const int u = blockIdx.x % U, rest = blockIdx.x / U;
        cg = a.CG - 1 - rest % a.CG;
        sp = rest / a.CG;
        i = u / a.g.H;
        h = u - i * a.g.H;
        r = kv_row(a.g, i);
    }
    // (uniform, which the compiler loses where the two ways meet)
    i = __builtin_amdgcn_readfirstlane(i);
    cg = __builtin_amdgcn_readfirstlane(cg);
    r = {__builtin_amdgcn_readfirstlane(r.e), __builtin_amdgcn_readfirstlane(r.pos), __builtin_amdgcn_readfirstlane(r.cnt)};
    const int u = i * a.g.H + h;
    const int all0 = cg * 64 * QT, c0 = all0 + w * 16 * QT;
    const KeyRange kr = key_range(a, r, all0, min(all0 + 64 * QT, a.N) - 1);
    const int start = (kr.beg & ~31) + sp * a.chunk, stop = min(kr.end, start + a.chunk);
    if (sp > 0 && start >= stop) return;
    const KeyRange own = c0 < a.N ? key_range(a, r, c0, min(c0 + 16 * QT, a.N) - 1) : KeyRange{0, 0, -1, 0};
    int lo[QT], hi[QT], col[QT];
    lane_columns<QT>(a, r, c0, li, col, lo, hi);
    TileSource src;
    {
        const long e = max(r.e, 0);
        src.k = a.g.codes + e * a.g.ce + (long)h * a.g.ch;
        src.v = src.k + a.g.ckv;
        src.ks = a.g.scales + e * a.g.se + (long)h * a.g.sh;
        src.vs = src.ks + a.g.skv;
    }
    WaveState<NB, BITS, T, QT> st;
    bool again = true;
    if constexpr (sizeof(T) == 2) again = wide_walk<NB, BITS, T, QT, true>(a, src, kr, own, start, stop, i, h, col, lo, hi, st, lds, lane, w);
    if (again) wide_walk<NB, BITS, T, QT, false>(a, src, kr, own, start, stop, i, h, col, lo, hi, st, lds, lane, w);
    store_columns<NB, BITS, T, QT>(a, st, u, i, h, sp, col, lo, hi, g);
}

// ------------------------------------------------------------------------------------------------
// One new position and one or two query heads per key head (NC columns): a matrix instruction would use 1 or 2 of its 16 columns
// and the wave would still pay for the terms and the transposition, so this form stays on the vector unit in fp32: a tile is 64
// keys, one a lane for the scores (the query's numbers come from LDS, the same address for all lanes), and one row of 16 lanes
// per 16 keys for the sum of the values (lane = 8 numbers, the weight of key i broadcast within the row by DPP).  About 360
// vector instructions per 64 keys at head_dim 96 against 1100 issue slots of the matrix form in fp32, and registers for four waves a
// SIMD: all 4096 waves of a 512-episode step are resident at once.  Measured against the matrix form (us, graph replay): 512 rows x
// 8 heads x 96, 32 positions, fp32 9.1 : 11.2; 64 x 8 x 128, 4096 positions, 4 bits, fp32 60 : 104, bf16 59 : 71, 8 bits 110 : 108
// (memory); two heads a key head, 64 x 16 / 8 x 128, 4096 positions, bf16 70 : 68, fp16 in 8 bits 105 : 123.
template <int NB, int BITS> struct VecTile {
    static constexpr int KW = 4 * NB * BITS / 4;                   // words of a whole row
    static constexpr int DV = RawTile<NB, BITS>::DV, VW = RawTile<NB, BITS>::VW;
    unsigned k[KW], ks, v[16][VW], vs[16];
};
template <int NB, int BITS> __device__ __forceinline__ void vec_load(VecTile<NB, BITS>& r, const TileSource& src, int k0, int rows, int lane) {
    constexpr int RB = 4 * NB * BITS, VB = VecTile<NB, BITS>::DV * BITS / 8;
    const int li = lane & 15, g = lane >> 4;
    const auto kc = rows_of<64>(src.k, k0, RB, rows), ks = rows_of<64>(src.ks, k0, 4, rows);
    buffer_words<RB>(kc, lane * RB, r.k);
    r.ks = __builtin_amdgcn_raw_buffer_load_b32(ks, lane * 4, 0, 0);
    const auto vc = rows_of<64>(src.v, k0, RB, rows), vs = rows_of<64>(src.vs, k0, 4, rows);
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
        const auto u = __builtin_amdgcn_raw_buffer_load_b128(vs, 64 * g + 4 * i, 0, 0);
        r.vs[i] = u[0]; r.vs[i + 1] = u[1]; r.vs[i + 2] = u[2]; r.vs[i + 3] = u[3];
    }
    const int vl = (NB == 3 ? min(li, 11) : li) * VB + 16 * g * RB;
#pragma unroll
    for (int i = 0; i < 16; ++i) buffer_words<VB>(vc, vl + i * RB, r.v[i]);
}

// two numbers (word w, pair j of it) as floats
template <int BITS> __device__ __forceinline__ f32x2 decode2(unsigned w, int j, float sc) {
    if constexpr (BITS == 4) {
        if (j == 0) return __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, sc, 0);
        if (j == 1) return __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, sc, 1);
        if (j == 2) return __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, sc, 2);
        return __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, sc, 3);
    } else {
        if (j == 0) return __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, sc, false);
        return __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, sc, true);
    }
}

// value of lane I of the row of 16 lanes, in every lane of the row
template <int I> __device__ __forceinline__ float row_lane(float v) { return __uint_as_float((unsigned)__builtin_amdgcn_mov_dpp((int)__float_as_uint(v), 0x150 + I, 0xF, 0xF, true)); }

template <int NB, int BITS, int NC, int I = 0>
__device__ __forceinline__ void vec_values(const VecTile<NB, BITS>& r, const float (&p)[NC], float (&acc)[NC][RawTile<NB, BITS>::DV], int block) {
    if constexpr (I < 16) {
        constexpr int DV = RawTile<NB, BITS>::DV, PPW = 16 / BITS;  // pairs a word
        const float sc = scale_of(r.vs[I], block);
        float w[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c) w[c] = row_lane<I>(p[c]);
#pragma unroll
        for (int j = 0; j < DV / 2; ++j) {
            const f32x2 y = decode2<BITS>(r.v[I][j / PPW], j % PPW, sc);
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                acc[c][2 * j] = __builtin_fmaf(w[c], y[0], acc[c][2 * j]);
                acc[c][2 * j + 1] = __builtin_fmaf(w[c], y[1], acc[c][2 * j + 1]);
            }
        }
        if constexpr (I % 4 == 3) __builtin_amdgcn_sched_barrier(0);
        vec_values<NB, BITS, NC, I + 1>(r, p, acc, block);
    }
}

// maximum / sum over the wave, vector instructions only: within a row of 16 by DPP, then over the four rows
__device__ __forceinline__ float dpp_xor1(float v) { return __uint_as_float((unsigned)__builtin_amdgcn_mov_dpp((int)__float_as_uint(v), 0xB1, 0xF, 0xF, true)); }
__device__ __forceinline__ float dpp_xor2(float v) { return __uint_as_float((unsigned)__builtin_amdgcn_mov_dpp((int)__float_as_uint(v), 0x4E, 0xF, 0xF, true)); }
__device__ __forceinline__ float dpp_half_mirror(float v) { return __uint_as_float((unsigned)__builtin_amdgcn_mov_dpp((int)__float_as_uint(v), 0x141, 0xF, 0xF, true)); }
__device__ __forceinline__ float dpp_mirror(float v) { return __uint_as_float((unsigned)__builtin_amdgcn_mov_dpp((int)__float_as_uint(v), 0x140, 0xF, 0xF, true)); }
__device__ __forceinline__ float all_max(float v) {
    v = fmaxf(v, dpp_xor1(v));
    v = fmaxf(v, dpp_xor2(v));
    v = fmaxf(v, dpp_half_mirror(v));
    v = fmaxf(v, dpp_mirror(v));
    return rows_max(v);
}
__device__ __forceinline__ float all_sum(float v) {
    v += dpp_xor1(v);
    v += dpp_xor2(v);
    v += dpp_half_mirror(v);
    v += dpp_mirror(v);
    return rows_sum(v);
}

template <int NB, int BITS, typename T, int NC>
__global__ __launch_bounds__(256, (NC == 1 && (BITS == 4 || NB <= 2) ? 4 : NC == 2 && BITS == 8 && NB >= 3 ? 2 : 3)) void attn_cache_vector_kernel(AttnCacheArgs a) {
    constexpr int D = 32 * NB, RB = 4 * NB * BITS, DV = RawTile<NB, BITS>::DV, KW = VecTile<NB, BITS>::KW, VW = VecTile<NB, BITS>::VW;
    constexpr int MROW = D + 4;
    __shared__ __attribute__((aligned(16))) unsigned char fresh_rows[4][2 * RB + 16];
    __shared__ __attribute__((aligned(16))) float queries[4][NC][D];
    __shared__ __attribute__((aligned(16))) float merge[4 * NC * MROW];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int li = lane & 15, g = lane >> 4;
    const int U = a.g.n * a.g.H;
    const int u = a.kw == 4 ? blockIdx.x % U : blockIdx.x * 4 + w, sp = a.kw == 4 ? blockIdx.x / U : 0;
    if (u >= U) return;                                            // (only with kw = 1: no barrier follows)
    const int i = u / a.g.H, h = u - i * a.g.H;
    const KvRow r = kv_row(a.g, i);
    const KeyRange kr = key_range(a, r, 0, a.N - 1);               // one step: every column sees the same keys
    const int start = (kr.beg & ~31) + sp * a.chunk, stop = min(kr.end, start + a.chunk);
    if (sp > 0 && start >= stop) return;                           // the whole workgroup: the item has fewer splits
    TileSource src;
    {
        const long e = max(r.e, 0);
        src.k = a.g.codes + e * a.g.ce + (long)h * a.g.ch;
        src.v = src.k + a.g.ckv;
        src.ks = a.g.scales + e * a.g.se + (long)h * a.g.sh;
        src.vs = src.ks + a.g.skv;
    }
    const int first = start + (a.kw == 4 ? 64 * w : 0), stride = a.kw * 64;
    VecTile<NB, BITS> raw;
    if (first < stop) vec_load<NB, BITS>(raw, src, first, stop - first, lane);

    // queries: 8 numbers a lane to LDS
    {
        const int c = lane >> 4, p = li;
        if (c < NC && p < 4 * NB) {
            float x[8];
            kv_load8<T>((const T*)a.q.p + (long)i * a.q.row + (long)(h * a.G + c) * a.q.head + 8 * p, a.q_vec, x);
#pragma unroll
            for (int e = 0; e < 8; e += 4) *(f32x4*)(&queries[w][c][8 * p + e]) = (f32x4){x[e], x[e + 1], x[e + 2], x[e + 3]};
        }
    }
    unsigned char* fr = fresh_rows[w];
    const int fresh_pos = append_row<NB, BITS, T>(a, r, i, h, sp, start, stop, kr.end, a.kw == 1 || w == 0, fr, lane);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();

    auto take_fresh = [&](int k0) {
        const int at = fresh_pos - k0;
        const unsigned ks = *(const unsigned*)(fr + 2 * RB), vs = *(const unsigned*)(fr + 2 * RB + 4);
#pragma unroll
        for (int q = 0; q < KW; q += 4) {                          // (read by all lanes, then selected: a read under the condition is a branch a word)
            const u32x4 x = *(const u32x4*)(fr + 4 * q);
#pragma unroll
            for (int e = 0; e < 4; ++e) raw.k[q + e] = lane == at ? x[e] : raw.k[q + e];
        }
        raw.ks = lane == at ? ks : raw.ks;
        constexpr int VB = DV * BITS / 8;
        unsigned vw[VW];
        lds_words<VB>(fr + RB + (NB == 3 ? min(li, 11) : li) * VB, vw);
#pragma unroll
        for (int q = 0; q < 16; ++q) {
            const bool here = 16 * g + q == at;
#pragma unroll
            for (int x = 0; x < VW; ++x) raw.v[q][x] = here ? vw[x] : raw.v[q][x];
            raw.vs[q] = here ? vs : raw.vs[q];
        }
    };
    float m[NC], l[NC], acc[NC][DV];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        m[c] = -INFINITY;
        l[c] = 0.f;
#pragma unroll
        for (int j = 0; j < DV; ++j) acc[c][j] = 0.f;
    }
    const int block = NB == 1 ? 0 : NB == 2 ? li >> 3 : li >> 2;
    for (int k0 = first; k0 < stop; k0 += stride) {
        if (fresh_pos >= k0 && fresh_pos < k0 + 64) take_fresh(k0);
        asm volatile("" ::: "memory");                             // the queries stay in LDS: held in registers across the loop they would cost 100 of them
        float s[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c) s[c] = 0.f;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const float sc = scale_of(raw.ks, b);
            float part[NC][2] = {};
#pragma unroll
            for (int q = 0; q < 8; ++q) {                          // four numbers at a time
                const int word = (32 * b + 4 * q) * BITS / 32, j0 = BITS == 4 ? (q & 1) * 2 : 0;
                const f32x2 y0 = decode2<BITS>(raw.k[word], j0, sc), y1 = decode2<BITS>(raw.k[word], j0 + 1, sc);
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const f32x4 x = *(const f32x4*)&queries[w][c][32 * b + 4 * q];
                    part[c][0] = __builtin_fmaf(y0[0], x[0], part[c][0]);
                    part[c][1] = __builtin_fmaf(y0[1], x[1], part[c][1]);
                    part[c][0] = __builtin_fmaf(y1[0], x[2], part[c][0]);
                    part[c][1] = __builtin_fmaf(y1[1], x[3], part[c][1]);
                }
            }
#pragma unroll
            for (int c = 0; c < NC; ++c) s[c] += part[c][0] + part[c][1];
            __builtin_amdgcn_sched_barrier(0);                     // (numbers decoded ahead of their use only fill registers)
        }
        const bool edge = k0 < kr.lo_all || k0 + 64 > stop;
        if (edge) {                                                // keys behind the end, and before the window: their value rows count as zeros
            const int key = k0 + lane;
#pragma unroll
            for (int c = 0; c < NC; ++c) s[c] = key >= kr.lo_all && key < stop ? s[c] : -INFINITY;
#pragma unroll
            for (int q = 0; q < 16; ++q) {
                const bool seen = k0 + 16 * g + q >= kr.lo_all;
                raw.vs[q] = seen ? raw.vs[q] : 0u;
#pragma unroll
                for (int x = 0; x < VW; ++x) raw.v[q][x] = seen ? raw.v[q][x] : 0u;
            }
        }
        float p[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            if (__any(__builtin_fmaf(s[c], a.c, -m[c] * a.c) > 8.f) || m[c] == -INFINITY) {       // (see tile_weights)
                const float mn = fmaxf(m[c], all_max(s[c]));
                const float corr = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m[c] - mn) * a.c);
                m[c] = mn;
                l[c] *= corr;
#pragma unroll
                for (int j = 0; j < DV; ++j) acc[c][j] *= corr;
            }
            const float mc = m[c] == -INFINITY ? 0.f : m[c] * a.c;
            p[c] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[c], a.c, -mc));
            l[c] += p[c];
        }
        __builtin_amdgcn_sched_barrier(0);
        vec_values<NB, BITS, NC>(raw, p, acc, block);
        if (k0 + stride < stop) vec_load<NB, BITS>(raw, src, k0 + stride, stop - k0 - stride, lane);
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        l[c] = all_sum(l[c]);
#pragma unroll
        for (int j = 0; j < DV; ++j) acc[c][j] = rows_sum(acc[c][j]);
    }
    const bool none = kr.beg >= kr.end;
    const int lanes = D / DV;                                      // lanes of the first row that hold the numbers: DV each
    if (a.kw == 1) {
        if (lane < lanes)
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const float inv = 1.0f / l[c];
                T* o = (T*)a.out.p + (long)i * a.out.row + (long)(h * a.G + c) * a.out.head + DV * lane;
                typedef __attribute__((ext_vector_type(DV))) T vt;
                vt v;
#pragma unroll
                for (int j = 0; j < DV; ++j) v[j] = kv_result<T>(none ? 0.f : acc[c][j] * inv);
                if constexpr (sizeof(vt) <= 16) *(vt*)o = v;
                else {
                    *(f32x4*)o = (f32x4){v[0], v[1], v[2], v[3]};
                    *(f32x4*)(o + 4) = (f32x4){v[4], v[5], v[6], v[7]};
                }
            }
        return;
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        float* mine = merge + (w * NC + c) * MROW;
        if (lane < lanes)
#pragma unroll
            for (int j = 0; j < DV; j += 2) *(f32x2*)(mine + DV * lane + j) = (f32x2){acc[c][j], acc[c][j + 1]};
        if (lane == 0) { mine[D] = m[c]; mine[D + 1] = l[c]; }
    }
    __syncthreads();
    for (int q = threadIdx.x; q < NC * (D / 4); q += 256) {
        const int c = q / (D / 4), d = (q % (D / 4)) * 4;
        float mx = -INFINITY, sum = 0.f;
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < 4; ++k) mx = fmaxf(mx, merge[(k * NC + c) * MROW + D]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float* from = merge + (k * NC + c) * MROW;
            const float f = from[D] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((from[D] - mx) * a.c);
            sum += from[D + 1] * f;
            o += *(const f32x4*)(from + d) * f;
        }
        if (a.nsplit == 1) {
            const float inv = 1.0f / sum;
            T* y = (T*)a.out.p + (long)i * a.out.row + (long)(h * a.G + c) * a.out.head + d;
            if constexpr (sizeof(T) == 4) {
                *(f32x4*)y = none ? (f32x4){0.f, 0.f, 0.f, 0.f} : o * inv;
            } else {
                typename Half16<T>::v4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = kv_result<T>(none ? 0.f : o[e] * inv);
                *(typename Half16<T>::v4*)y = v;
            }
        } else {
            float* y = a.part + (((long)sp * U + u) * a.N + c) * (D + 2);
            *(f32x2*)(y + d) = (f32x2){o[0], o[1]};
            *(f32x2*)(y + d + 2) = (f32x2){o[2], o[3]};
            if (d == 0) *(f32x2*)(y + D) = (f32x2){mx, sum};
        }
    }
}

// The splits of one column put together.  WV waves take one column; D / 4 lanes read one split's numbers, so several splits are in
// flight at a time (read one after the other by one wave, 32 splits cost 15 us of memory round trips; four waves: 4 us).
template <typename T, int NB, int WV>
__global__ __launch_bounds__(256) void attn_cache_join_kernel(AttnCacheArgs a, int cols_per_group) {
    constexpr int D = 32 * NB, LPS = D / 4, PAR = 64 * WV / LPS, CPB = 4 / WV;       // lanes per split, splits at a time, columns a workgroup
    __shared__ __attribute__((aligned(16))) f32x4 sums[CPB][PAR][LPS];
    __shared__ float red[4], ls[CPB][PAR];
    const int U = a.g.n * a.g.H;
    const int tid = threadIdx.x % (64 * WV), cw = threadIdx.x / (64 * WV);
    const int item = blockIdx.x * CPB + cw;
    const bool live = item < U * a.N;
    const int u = live ? item / a.N : 0, c = live ? item - u * a.N : 0;
    const int i = u / a.g.H, h = u - i * a.g.H, step = c / a.G, hq = h * a.G + c - step * a.G;
    const KvRow r = kv_row(a.g, i);
    const int c0 = c / cols_per_group * cols_per_group;
    const KeyRange kr = key_range(a, r, c0, min(c0 + cols_per_group, a.N) - 1);
    const KeyRange own = key_range(a, r, c, c);
    const int ns = max((kr.end - (kr.beg & ~31) + a.chunk - 1) / a.chunk, 1);       // splits that this column's group really has
    const long hop = (long)U * a.N * (D + 2);
    const float* base = a.part + ((long)u * a.N + c) * (D + 2);
    const int q = tid % LPS, w = tid / LPS;
    float m = -INFINITY;
    for (int s = tid; s < ns; s += 64 * WV) m = fmaxf(m, base[s * hop + D]);
    m = wave_max(m);
    if constexpr (WV > 1) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
        __syncthreads();
        m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    }
    float l = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    if (w < PAR) {
#pragma unroll 4
        for (int s = w; s < ns; s += PAR) {
            const float* y = base + s * hop;
            const f32x2 v0 = *(const f32x2*)(y + 4 * q), v1 = *(const f32x2*)(y + 4 * q + 2), ml = *(const f32x2*)(y + D);
            const float f = ml[0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((ml[0] - m) * a.c);
            l += ml[1] * f;
            o += (f32x4){v0[0], v0[1], v1[0], v1[1]} * f;
        }
        sums[cw][w][q] = o;
        if (q == 0) ls[cw][w] = l;
    }
    __syncthreads();
    if (tid >= LPS || !live) return;
    const int parts = min(PAR, ns);
    o = sums[cw][0][tid];
    l = ls[cw][0];
    for (int k = 1; k < parts; ++k) {                              // fixed order
        o += sums[cw][k][tid];
        l += ls[cw][k];
    }
    const bool none = own.beg >= own.end;
    const float inv = 1.0f / l;
    T* y = (T*)a.out.p + (long)i * a.out.row + (long)step * a.out.step + (long)hq * a.out.head + 4 * tid;
    if constexpr (sizeof(T) == 4) {
        *(f32x4*)y = none ? (f32x4){0.f, 0.f, 0.f, 0.f} : o * inv;
    } else {
        typename Half16<T>::v4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = kv_result<T>(none ? 0.f : o[e] * inv);
        *(typename Half16<T>::v4*)y = v;
    }
}

template <typename T, int NB> void launch_join(const AttnCacheArgs& a, int cols, hipStream_t s) {
    const unsigned items = (unsigned)(a.g.n * a.g.H * a.N);         // (splits are made for at most 4096 items of at most 128 columns)
    if (a.nsplit <= 8) hipLaunchKernelGGL((attn_cache_join_kernel<T, NB, 1>), dim3((items + 3) / 4), dim3(256), 0, s, a, cols);
    else hipLaunchKernelGGL((attn_cache_join_kernel<T, NB, 4>), dim3(items), dim3(256), 0, s, a, cols);
}

template <int NB, int BITS, typename T, int QT>
int launch_wide(const AttnCacheArgs& a, unsigned blocks, hipStream_t s) {
    constexpr int lds = 2 * WideTile<NB, BITS>::bytes;
    if (int rc = otter_reserve_lds((const void*)attn_cache_wide_kernel<NB, BITS, T, QT>, lds, "otter_attn_cache")) return rc;
    hipLaunchKernelGGL((attn_cache_wide_kernel<NB, BITS, T, QT>), dim3(blocks), dim3(256), lds, s, a);
    return OTTER_OK;
}

template <int NB, int BITS, typename T>
int launch_qt(const AttnCacheArgs& a, int qt, unsigned blocks, hipStream_t s) {
    if (a.vec) {
        if (a.G == 1) hipLaunchKernelGGL((attn_cache_vector_kernel<NB, BITS, T, 1>), dim3(blocks), dim3(256), 0, s, a);
        else hipLaunchKernelGGL((attn_cache_vector_kernel<NB, BITS, T, 2>), dim3(blocks), dim3(256), 0, s, a);
        return OTTER_OK;
    }
    if (a.wide) {
        if constexpr (wide_columns(KvElem<T>::code, NB) == 2)
            if (qt == 2) return launch_wide<NB, BITS, T, 2>(a, blocks, s);
        return launch_wide<NB, BITS, T, 1>(a, blocks, s);
    }
    if constexpr (narrow_columns(KvElem<T>::code, NB) == 2)
        if (qt == 2) {
            hipLaunchKernelGGL((attn_cache_kernel<NB, BITS, T, 2>), dim3(blocks), dim3(256), 0, s, a);
            return OTTER_OK;
        }
    hipLaunchKernelGGL((attn_cache_kernel<NB, BITS, T, 1>), dim3(blocks), dim3(256), 0, s, a);
    return OTTER_OK;
}

template <typename T, int BITS> int launch_nb(const AttnCacheArgs& a, int nb, int qt, unsigned blocks, hipStream_t s) {
    if (nb == 1) return launch_qt<1, BITS, T>(a, qt, blocks, s);
    if (nb == 2) return launch_qt<2, BITS, T>(a, qt, blocks, s);
    if (nb == 3) return launch_qt<3, BITS, T>(a, qt, blocks, s);
    return launch_qt<4, BITS, T>(a, qt, blocks, s);
}

}  // namespace

template <typename T> int otter_attn_cache_launch(const AttnCacheArgs& a, int nb, int bits, int qt, unsigned blocks, hipStream_t s) {
    if (int rc = bits == 4 ? launch_nb<T, 4>(a, nb, qt, blocks, s) : launch_nb<T, 8>(a, nb, qt, blocks, s)) return rc;
    OTTER_CHECK_LAUNCH("otter_attn_cache");
    if (a.nsplit > 1) {
        const int cols = (a.wide ? 64 : 16) * qt;
        if (nb == 1) launch_join<T, 1>(a, cols, s);
        else if (nb == 2) launch_join<T, 2>(a, cols, s);
        else if (nb == 3) launch_join<T, 3>(a, cols, s);
        else launch_join<T, 4>(a, cols, s);
        OTTER_CHECK_LAUNCH("otter_attn_cache (join)");
    }
    return OTTER_OK;
}
#endif
