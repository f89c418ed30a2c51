// Attention over the quantised K/V cache (kv_cache.hpp): flash form, one or many new positions a row, grouped heads.
//
//   out[t, h] = sum_j p_j v_j / sum_j p_j,   p_j = 2^(c (q . k_j) - m),   c = scale log2 e,   m = running maximum of c (q . k_j),
// over the cached positions j that query t of the row sees.
//
// Operands.  A stored number has at most 4 significant bits, so k_j and v_j are exact in bf16 and the products run on
// v_mfma_f32_16x16x32_bf16 with fp32 accumulation.  q and p are written as sums of bf16 terms: q exactly (1 term for bf16, 2 for
// fp16, 3 for fp32), p in 2 terms (2^-17 relative, far below the output's own rounding) for 16-bit and 3 (2^-24) for fp32 outputs.
//
// Tile.  A wave owns 16 * QT columns (query positions x heads of one key head's group) and walks over tiles of 32 keys, all
// state in registers.  S^T = K Q^T puts 8 scores of one column in a lane, keys 4g+i and 16+4g+i (g = lane / 16), which is the
// B operand of out^T = V^T P^T if V's rows are taken in the same key order: no exchange between lanes.  K is loaded as it lies
// (lane = key, head_dim / 4 consecutive numbers), V as 8 rows x head_dim / 16 numbers a lane and turned by v_perm after the
// conversion.  Rows past the last key are never read (addresses are cut at it).
//
// Masked keys.  Scores are selected, but 0 * NaN of a masked value row would still reach the accumulator.  The fast pass ignores
// that; if a wave ends with a non-finite accumulator it runs again with the value rows cleaned and NaN set where a row that the
// column really sees is not finite.
#pragma once
#include "kv_cache.hpp"

struct AttnCacheArgs {
    KvGeom g;
    KvOperand<const void> q; int q_vec;
    KvOperand<void> out;
    KvOperand<const void> kn, vn; int new_vec;      // fresh key / value rows to append (null: the cache is complete)
    int G, N, CG;                                   // query heads per key head, columns T * G, column groups of 16 * QT
    int causal, window, max_len;
    float c;
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

// host: instantiated per element type (attn_cache_*.hip)
template <typename T> int otter_attn_cache_launch(const AttnCacheArgs& a, int nb, int bits, int qt, unsigned blocks, hipStream_t s);

#ifdef OTTER_ATTN_CACHE_IMPL
namespace {

typedef __attribute__((ext_vector_type(4))) unsigned u32x4;
typedef __attribute__((ext_vector_type(4), aligned(4))) unsigned u32x4_a4;     // 16 bytes at a 4-byte boundary

// what one tile of 32 keys needs from memory, as loaded
template <int NB, int BITS> struct RawTile {
    static constexpr int KW = NB * BITS / 4;                       // words of one key a lane holds (a quarter of its row)
    static constexpr int DV = NB == 3 ? 8 : 2 * NB;                // numbers of a value row a lane holds (NB = 3: 12 of 16 lanes, 8 each)
    static constexpr int VW = DV * BITS / 8 > 4 ? 2 : 1;           // words of those
    unsigned k[2][KW], v[8][VW];
    unsigned ks[2], vs[8];                                         // scale words of the rows
};

template <int NB, int BITS> struct TileSource {
    const unsigned char* kc; const unsigned char* vc;              // rows of this episode and head
    const unsigned char* ksc; const unsigned char* vsc;
};

__device__ __forceinline__ int v_row(int g, int i) { return 4 * g + (i & 3) + 16 * (i >> 2); }   // key of element i of lane group g's operand

template <int W> __device__ __forceinline__ void load_words(const unsigned char* p, unsigned (&w)[W]) {
    if constexpr (W == 1) w[0] = *(const unsigned*)p;
    else if constexpr (W == 2) { const uint2 u = *(const uint2*)p; w[0] = u.x; w[1] = u.y; }
    else if constexpr (W == 3) {
        typedef __attribute__((ext_vector_type(3), aligned(4))) unsigned u3;
        const u3 u = *(const u3*)p;
        w[0] = u[0]; w[1] = u[1]; w[2] = u[2];
    } else if constexpr (W == 6) {
#pragma unroll
        for (int i = 0; i < 3; ++i) { const uint2 u = *(const uint2*)(p + 8 * i); w[2 * i] = u.x; w[2 * i + 1] = u.y; }
    } else {
#pragma unroll
        for (int i = 0; i < W / 4; ++i) {
            const u32x4 u = *(const u32x4*)(p + 16 * i);
            w[4 * i] = u[0]; w[4 * i + 1] = u[1]; w[4 * i + 2] = u[2]; w[4 * i + 3] = u[3];
        }
    }
}
template <int BYTES, int W> __device__ __forceinline__ void load_part(const unsigned char* p, unsigned (&w)[W]) {
    if constexpr (BYTES == 1) w[0] = *p;
    else if constexpr (BYTES == 2) w[0] = *(const unsigned short*)p;
    else load_words<W>(p, w);
}

// rows k0 .. k0 + 31 of the cache; TAIL: only nk of them exist, the others repeat the last one
template <int NB, int BITS, bool TAIL>
__device__ __forceinline__ void load_tile(RawTile<NB, BITS>& r, const TileSource<NB, BITS>& src, int k0, int nk, int lane) {
    constexpr int RB = 4 * NB * BITS, KB = RB / 4, DV = RawTile<NB, BITS>::DV, VB = DV * BITS / 8;
    const int li = lane & 15, g = lane >> 4;
    const unsigned char* kc = src.kc + (long)k0 * RB;
    const unsigned char* vc = src.vc + (long)k0 * RB;
    const unsigned char* ksc = src.ksc + (long)k0 * 4;
    const unsigned char* vsc = src.vsc + (long)k0 * 4;
    const int vl = NB == 3 ? min(li, 11) * VB : li * VB;           // NB = 3: lanes 12 .. 15 repeat lane 11 (their output rows are not stored)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int row = TAIL ? min(li + 16 * h, nk - 1) : li + 16 * h;
        load_words(kc + row * RB + g * KB, r.k[h]);
        r.ks[h] = *(const unsigned*)(ksc + row * 4);
    }
    if constexpr (TAIL) {
#pragma unroll
        for (int i = 0; i < 8; ++i) r.vs[i] = *(const unsigned*)(vsc + min(v_row(g, i), nk - 1) * 4);
    } else {
        const u32x4_a4 a = *(const u32x4_a4*)(vsc + 16 * g), b = *(const u32x4_a4*)(vsc + 64 + 16 * g);
#pragma unroll
        for (int i = 0; i < 4; ++i) { r.vs[i] = a[i]; r.vs[4 + i] = b[i]; }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) load_part<VB>(vc + (TAIL ? min(v_row(g, i), nk - 1) : v_row(g, i)) * RB + vl, r.v[i]);
}

// scale operand of a block conversion: the wanted byte moved to the exponent's place (the conversion reads nothing else)
__device__ __forceinline__ float scale_of(unsigned word, int block) {
    const unsigned rot = (unsigned)(9 + 8 * block) & 31u;         // rotate right by 9 + 8 b: byte b lands on bits 23 .. 30
    return __uint_as_float(__builtin_amdgcn_alignbit(word, word, rot));
}

// eight consecutive codes (from word w of a lane's row part on) as bf16
template <int BITS> __device__ __forceinline__ bf16x8 decode8(const unsigned* w, float sc) {
    bf16x2 d[4];
    if constexpr (BITS == 4) {
        d[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], sc, 0);
        d[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], sc, 1);
        d[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], sc, 2);
        d[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], sc, 3);
    } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            d[2 * h] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[h], sc, false);
            d[2 * h + 1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[h], sc, true);
        }
    }
    bf16x8 o;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = d[i >> 1][i & 1];
    return o;
}
// pair number j of a lane's part of a value row
template <int BITS> __device__ __forceinline__ unsigned decode_pair(const unsigned* w, int j, float sc) {
    bf16x2 d;
    if constexpr (BITS == 4) {
        if (j == 0) d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], sc, 0);
        else if (j == 1) d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], sc, 1);
        else if (j == 2) d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], sc, 2);
        else d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], sc, 3);
    } else {
        if (j & 1) d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[j >> 1], sc, true);
        else d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[j >> 1], sc, false);
    }
    return __builtin_bit_cast(unsigned, d);
}

__device__ __forceinline__ unsigned pack_bf16(float a, float b) {
    return __builtin_bit_cast(unsigned, (bf16x2){(__bf16)a, (__bf16)b});
}

// eight numbers as NP bf16 operands whose sum they are (to 2^-8 of the last term)
template <int NP> __device__ __forceinline__ void split_p(const float (&p)[8], bf16x8 (&out)[NP]) {
    unsigned w[NP][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float a = p[2 * i], b = p[2 * i + 1];
#pragma unroll
        for (int n = 0; n < NP; ++n) {
            w[n][i] = pack_bf16(a, b);
            if (n + 1 < NP) {
                a -= __uint_as_float(w[n][i] << 16);
                b -= __uint_as_float(w[n][i] & 0xffff0000u);
            }
        }
    }
#pragma unroll
    for (int n = 0; n < NP; ++n) {
        const u32x4 v = {w[n][0], w[n][1], w[n][2], w[n][3]};
        out[n] = __builtin_bit_cast(bf16x8, v);
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

template <int NB, int BITS, typename T, int QT, bool CAREFUL>
__device__ __forceinline__ void tile_step(const RawTile<NB, BITS>& r, WaveState<NB, BITS, T, QT>& st, const bf16x8 (&qf)[QT][AttnTerms<T>::q][NB],
                                          int k0, bool masked, const int (&lo)[QT], const int (&hi)[QT], float c, int lane) {
    constexpr int NQ = AttnTerms<T>::q, NP = AttnTerms<T>::p, DV = RawTile<NB, BITS>::DV;
    const int li = lane & 15, g = lane >> 4;
    f32x4 s[QT][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        bf16x8 kf[NB];
#pragma unroll
        for (int j = 0; j < NB; ++j)                               // unit NB g + j of 8 numbers lies in block (NB g + j) / 4
            kf[j] = decode8<BITS>(&r.k[h][j * BITS / 4], scale_of(r.ks[h], NB == 1 ? 0 : NB == 2 ? g >> 1 : NB == 4 ? g : (3 * g + j) >> 2));
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            s[t][h] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int n = NQ - 1; n >= 0; --n)                      // small terms first
#pragma unroll
                for (int j = 0; j < NB; ++j) s[t][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[j], qf[t][n][j], s[t][h], 0, 0, 0);
        }
    }
    // value rows: 8 keys x DV numbers a lane -> DV operands of 8 keys
    u32x4 vf[DV];
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const int block = NB == 1 ? 0 : NB == 2 ? li >> 3 : li >> 2;
        const float s0 = scale_of(r.vs[i], block), s1 = scale_of(r.vs[i + 1], block);
#pragma unroll
        for (int j = 0; j < DV / 2; ++j) {
            const unsigned a = decode_pair<BITS>(r.v[i], j, s0), b = decode_pair<BITS>(r.v[i + 1], j, s1);
            vf[2 * j][i >> 1] = __builtin_amdgcn_perm(b, a, 0x05040100u);
            vf[2 * j + 1][i >> 1] = __builtin_amdgcn_perm(b, a, 0x07060302u);
        }
    }
    bf16x8 bad[CAREFUL ? DV : 1];
    if constexpr (CAREFUL) {
#pragma unroll
        for (int j = 0; j < DV; ++j) {
            u32x4 flag;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const unsigned w = vf[j][i];
                const bool x0 = (w & 0x7f80u) == 0x7f80u, x1 = (w & 0x7f800000u) == 0x7f800000u;
                flag[i] = (x0 ? 0x3f80u : 0u) | (x1 ? 0x3f800000u : 0u);
                vf[j][i] = w & ~((x0 ? 0xffffu : 0u) | (x1 ? 0xffff0000u : 0u));
            }
            bad[j] = __builtin_bit_cast(bf16x8, flag);
        }
    }
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = s[t][i >> 2][i & 3];
        if (masked) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int key = k0 + v_row(g, i);
                x[i] = (key <= hi[t] && key >= lo[t]) ? x[i] : -INFINITY;
            }
        }
        float mx = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
        mx = rows_max(mx);
        const float mn = fmaxf(st.m[t], mx);
        const float mc = mn == -INFINITY ? 0.f : mn * c;
        if (__any(mn > st.m[t])) {
            const float corr = __builtin_amdgcn_exp2f(st.m[t] * c - mc);
            st.l[t] *= corr;
#pragma unroll
            for (int j = 0; j < DV; ++j) st.acc[t][j] *= corr;
        }
        st.m[t] = mn;
        float p[8];
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], c, -mc));
            sum += p[i];
        }
        st.l[t] += sum;
        bf16x8 pf[NP];
        split_p<NP>(p, pf);
#pragma unroll
        for (int n = NP - 1; n >= 0; --n)
#pragma unroll
            for (int j = 0; j < DV; ++j)
                st.acc[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, vf[j]), pf[n], st.acc[t][j], 0, 0, 0);
        if constexpr (CAREFUL) {
            u32x4 seen;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int k1 = k0 + v_row(g, 2 * i), k2 = k0 + v_row(g, 2 * i + 1);
                seen[i] = (k1 <= hi[t] && k1 >= lo[t] ? 0x3f80u : 0u) | (k2 <= hi[t] && k2 >= lo[t] ? 0x3f800000u : 0u);
            }
#pragma unroll
            for (int j = 0; j < DV; ++j) {
                f32x4 n = {0.f, 0.f, 0.f, 0.f};
                n = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bad[j], __builtin_bit_cast(bf16x8, seen), n, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; ++i) st.acc[t][j][i] = n[i] > 0.f ? __builtin_nanf("") : st.acc[t][j][i];
            }
        }
    }
}

// the fresh row of position `pos` in place of what the cache still holds there
template <int NB, int BITS>
__device__ __forceinline__ void take_fresh(RawTile<NB, BITS>& r, const unsigned char* fresh, int k0, int pos, int lane) {
    constexpr int RB = 4 * NB * BITS, KB = RB / 4, DV = RawTile<NB, BITS>::DV, VB = DV * BITS / 8, KW = RawTile<NB, BITS>::KW, VW = RawTile<NB, BITS>::VW;
    const int li = lane & 15, g = lane >> 4;
    unsigned kw[KW], vw[VW];
#pragma unroll
    for (int i = 0; i < KW; ++i) kw[i] = *(const unsigned*)(fresh + g * KB + 4 * i);
    load_part<VB>(fresh + RB + (NB == 3 ? min(li, 11) : li) * VB, vw);
    const unsigned ks = *(const unsigned*)(fresh + 2 * RB), vs = *(const unsigned*)(fresh + 2 * RB + 4);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const bool here = k0 + li + 16 * h == pos;
#pragma unroll
        for (int i = 0; i < KW; ++i) r.k[h][i] = here ? kw[i] : r.k[h][i];
        r.ks[h] = here ? ks : r.ks[h];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const bool here = k0 + v_row(g, i) == pos;
#pragma unroll
        for (int w = 0; w < VW; ++w) r.v[i][w] = here ? vw[w] : r.v[i][w];
        r.vs[i] = here ? vs : r.vs[i];
    }
}

// Items: (split, row, key head, column group).  A workgroup of four waves takes one item with the keys dealt out in tiles
// (kw = 4), or four items: neighbouring column groups of one (row, head), which read the same rows, or, with one column
// group, four (row, head) pairs.  (row, head) runs fastest over the workgroups, so that the column groups of one pair meet in
// one XCD's L2; the last column groups, which see the most keys under a causal mask, start first.
template <int NB, int BITS, typename T, int QT>
__global__ __launch_bounds__(256) void attn_cache_kernel(AttnCacheArgs a) {
    constexpr int D = 32 * NB, RB = 4 * NB * BITS, DV = RawTile<NB, BITS>::DV, NQ = AttnTerms<T>::q;
    constexpr int MROW = D + 4;                                    // padded row of the merge buffer
    __shared__ __attribute__((aligned(16))) unsigned char fresh_rows[4][2 * RB + 16];
    __shared__ float merge[4 * 16 * MROW];
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

    // columns of this lane
    int lo[QT], hi[QT], col[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        col[t] = c0 + 16 * t + li;
        const int step = col[t] / a.G;
        const int qp = a.causal ? r.pos + step : r.pos + r.cnt - 1;
        hi[t] = (col[t] < a.N && step < r.cnt && r.e >= 0) ? min(min(qp, a.g.S - 1), a.max_len - 1) : -1;
        lo[t] = a.window ? max(qp - a.window + 1, 0) : 0;
    }

    // the fresh row: codes to the cache and, for this wave's own tiles, to LDS
    unsigned char* fr = fresh_rows[w];
    int fresh_pos = -1;
    // (a position that max_len hides is stored all the same, by the first split)
    const bool sees_fresh = r.pos >= start && r.pos < stop;
    if (a.kn.p && r.e >= 0 && (sees_fresh || (sp == 0 && r.pos >= kr.end && r.pos < a.g.S))) {
        fresh_pos = sees_fresh ? r.pos : -1;
        int from = i;                                              // an episode listed twice: the last listing is the one that is stored and seen
        if (a.g.idx) {
            int last = i;
            for (int j = i + 1 + lane; j < a.g.n; j += 64) last = a.g.idx[j] == r.e ? j : last;
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) last = max(last, __shfl_xor(last, o, 64));
            from = __builtin_amdgcn_readfirstlane(last);
        }
        const int kv = lane >> 4, p = li;                          // lanes 0 .. 15: the key row, 16 .. 31: the value row, 8 numbers each
        float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        const bool on = lane < 32 && p < 4 * NB;
        if (on) {
            const KvOperand<const void>& o = kv ? a.vn : a.kn;
            kv_load8<T>((const T*)o.p + (long)from * o.row + (long)h * o.head + 8 * p, a.new_vec, x);
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
            // one wave of the item writes the row: the first of the group with key 0's columns
            if (from == i && cg == 0 && (a.kw == 1 || w == 0)) {
                unsigned char* cc = a.g.codes + kv * a.g.ckv + (long)r.e * a.g.ce + (long)h * a.g.ch + (long)r.pos * RB + p * BITS;
                if constexpr (BITS == 4) *(unsigned*)cc = cw[0];
                else *(uint2*)cc = make_uint2(cw[0], cw[BITS / 4 - 1]);
                if ((p & 3) == 0) a.g.scales[kv * a.g.skv + (long)r.e * a.g.se + (long)h * a.g.sh + (long)r.pos * 4 + (p >> 2)] = (unsigned char)sb;
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }

    // query operands: numbers 8 NB g + 8 j .. + 7 of the lane's column, as a sum of bf16 terms (cut, not rounded: the rest is exact)
    bf16x8 qf[QT][NQ][NB];
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
                    const float cut = __uint_as_float(__float_as_uint(rest) & 0xffff0000u);
                    qf[t][n][j][e] = (__bf16)cut;
                    rest -= cut;
                }
            }
        }
    }

    TileSource<NB, BITS> src;
    {
        const long e = max(r.e, 0);
        src.kc = a.g.codes + e * a.g.ce + (long)h * a.g.ch;
        src.vc = src.kc + a.g.ckv;
        src.ksc = a.g.scales + e * a.g.se + (long)h * a.g.sh;
        src.vsc = src.ksc + a.g.skv;
    }
    WaveState<NB, BITS, T, QT> st;
    const int first = start + (a.kw == 4 ? 32 * w : 0), stride = a.kw * 32;
    auto load = [&](RawTile<NB, BITS>& raw, int k0) {
        if (k0 + 32 <= stop) load_tile<NB, BITS, false>(raw, src, k0, 32, lane);
        else load_tile<NB, BITS, true>(raw, src, k0, stop - k0, lane);
        if (fresh_pos >= k0 && fresh_pos < k0 + 32) take_fresh<NB, BITS>(raw, fr, k0, fresh_pos, lane);
    };
    auto walk = [&](auto careful) {
        st.reset();
        if (first >= stop) return;
        RawTile<NB, BITS> cur, nxt;
        load(cur, first);
        for (int k0 = first; k0 < stop; k0 += stride) {
            const bool more = k0 + stride < stop;
            if (more) load(nxt, k0 + stride);
            const bool masked = decltype(careful)::value || k0 + 31 > kr.hi_all || k0 + 31 >= stop || k0 < kr.lo_all;
            tile_step<NB, BITS, T, QT, decltype(careful)::value>(cur, st, qf, k0, masked, lo, hi, a.c, lane);
            if (more) cur = nxt;
        }
    };
    walk(std::integral_constant<bool, false>{});
    {
        float z = 0.f;
#pragma unroll
        for (int t = 0; t < QT; ++t)
#pragma unroll
            for (int j = 0; j < DV; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) z = __builtin_fmaf(st.acc[t][j][e], 0.f, z);
        if (__any(!(z == 0.f))) walk(std::integral_constant<bool, true>{});
    }
#pragma unroll
    for (int t = 0; t < QT; ++t) st.l[t] = rows_sum(st.l[t]);

    const long part_row = ((long)sp * U + u) * a.N;
    if (a.kw == 1) {                                               // the lane holds numbers 4 DV g .. + 4 DV - 1 of its column
        if (NB == 3 && g == 3) return;
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            if (col[t] >= a.N) continue;
            const int step = col[t] / a.G, hq = h * a.G + col[t] - step * a.G;
            const float inv = lo[t] <= hi[t] ? 1.0f / st.l[t] : 0.f;
            T* o = (T*)a.out.p + (long)i * a.out.row + (long)step * a.out.step + (long)hq * a.out.head + 4 * DV * g;
            const bool none = lo[t] > hi[t];
#pragma unroll
            for (int q = 0; q < DV / 2; ++q) {                     // 8 consecutive numbers: rows 8 / DV at a time
                float y[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) { const int d = 8 * q + e; y[e] = none ? 0.f : st.acc[t][d % DV][d / DV] * inv; }
                if constexpr (sizeof(T) == 4) {
                    *(f32x4*)(o + 8 * q) = (f32x4){y[0], y[1], y[2], y[3]};
                    *(f32x4*)(o + 8 * q + 4) = (f32x4){y[4], y[5], y[6], y[7]};
                } else {
                    typename Half16<T>::v8 v;
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = (T)y[e];
                    *(typename Half16<T>::v8*)(o + 8 * q) = v;
                }
            }
        }
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
                    for (int e = 0; e < 4; ++e) v[e] = (T)(none ? 0.f : o[e] * inv);
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

// the splits of one column put together: one wave a column, D / 64 (rounded up) numbers a lane
template <typename T>
__global__ __launch_bounds__(256) void attn_cache_join_kernel(AttnCacheArgs a, int D, int cols_per_group) {
    const int lane = threadIdx.x & 63;
    const long item = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int U = a.g.n * a.g.H;
    if (item >= (long)U * a.N) return;
    const int u = (int)(item / a.N), c = (int)(item - (long)u * a.N);
    const int i = u / a.g.H, h = u - i * a.g.H, step = c / a.G, hq = h * a.G + c - step * a.G;
    const KvRow r = kv_row(a.g, i);
    const int c0 = c / cols_per_group * cols_per_group;
    const KeyRange kr = key_range(a, r, c0, min(c0 + cols_per_group, a.N) - 1);
    const KeyRange own = key_range(a, r, c, c);
    const bool none = own.beg >= own.end;
    const int span = kr.end - (kr.beg & ~31);
    const int ns = max((span + a.chunk - 1) / a.chunk, 1);
    const long hop = (long)U * a.N * (D + 2);
    const float* base = a.part + ((long)u * a.N + c) * (D + 2);
    float m = -INFINITY;
    for (int s = lane; s < ns; s += 64) m = fmaxf(m, base[s * hop + D]);
    m = wave_max(m);
    float l = 0.f, o0 = 0.f, o1 = 0.f;
#pragma unroll 4
    for (int s = 0; s < ns; ++s) {
        const float* y = base + s * hop;
        const float ms = y[D], f = ms == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((ms - m) * a.c);
        l += y[D + 1] * f;
        if (2 * lane < D) {
            const f32x2 v = *(const f32x2*)(y + 2 * lane);
            o0 += v[0] * f;
            o1 += v[1] * f;
        }
    }
    if (2 * lane >= D) return;
    const float inv = 1.0f / l;
    T* y = (T*)a.out.p + (long)i * a.out.row + (long)step * a.out.step + (long)hq * a.out.head + 2 * lane;
    y[0] = (T)(none ? 0.f : o0 * inv);
    y[1] = (T)(none ? 0.f : o1 * inv);
}

template <int NB, int BITS, typename T>
void launch_qt(const AttnCacheArgs& a, int qt, unsigned blocks, hipStream_t s) {
    if (qt == 1) hipLaunchKernelGGL((attn_cache_kernel<NB, BITS, T, 1>), dim3(blocks), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((attn_cache_kernel<NB, BITS, T, 2>), dim3(blocks), dim3(256), 0, s, a);
}

template <typename T, int BITS> void launch_nb(const AttnCacheArgs& a, int nb, int qt, unsigned blocks, hipStream_t s) {
    if (nb == 1) launch_qt<1, BITS, T>(a, qt, blocks, s);
    else if (nb == 2) launch_qt<2, BITS, T>(a, qt, blocks, s);
    else if (nb == 3) launch_qt<3, BITS, T>(a, qt, blocks, s);
    else launch_qt<4, BITS, T>(a, qt, blocks, s);
}

}  // namespace

template <typename T> int otter_attn_cache_launch(const AttnCacheArgs& a, int nb, int bits, int qt, unsigned blocks, hipStream_t s) {
    if (bits == 4) launch_nb<T, 4>(a, nb, qt, blocks, s);
    else launch_nb<T, 8>(a, nb, qt, blocks, s);
    OTTER_CHECK_LAUNCH("otter_attn_cache");
    if (a.nsplit > 1) {
        const long items = (long)a.g.n * a.g.H * a.N;
        hipLaunchKernelGGL(attn_cache_join_kernel<T>, dim3((unsigned)((items + 3) / 4)), dim3(256), 0, s, a, 32 * nb, 16 * qt);
        OTTER_CHECK_LAUNCH("otter_attn_cache (join)");
    }
    return OTTER_OK;
}
#endif
