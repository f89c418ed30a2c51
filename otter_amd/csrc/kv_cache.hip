// Writing the quantised K/V cache and reading it back (layout and arithmetic: kv_cache.hpp).
#include <algorithm>

#include "kv_cache.hpp"

namespace {

// Both kernels move 8 numbers a lane and piece: a lane's codes are 4 (or 8) bytes, four lanes share a block and its scale.  Lanes
// run along the head dimension (a row takes 4, 8 or 16 lanes; with head_dim 96 four of the 16 idle), then along the steps, then
// along the heads: a cache row is contiguous with the row of the next step, so a wave's codes form one run, and its numbers runs
// of head_dim elements.  Memory-bound: head_dim * (element size + BITS / 8) + 4 bytes a row, no reuse; a lane takes up to four
// pieces whose loads are requested together, and the four scale bytes of a row leave in one store.  16 x 4093 steps x 8 heads of
// 128 between bf16 and 4 bits, 339 MB: write 63 us on the same numbers again, 73 on others each time (4.6 TB/s), 90 behind a read-back, whose 268 MB
// of results fill the last-level cache (256 MB) and have to leave it; read 55 us (6.1 TB/s: the codes, 71 MB, stay in that cache).  24 x 6001 x 8 heads of 64,
// fp16, 373 MB: 78 and 71 us.  Copies reach 7.0 TB/s of 2 x 128 MB (inside the cache), 5.4 of 2 x 256 MB and 4.8 of 2 x 2 GB.
template <int NB> struct RowLanes { static constexpr int P = NB == 1 ? 4 : NB == 2 ? 8 : 16, live = 4 * NB; };

template <int NB, int BITS, typename T, int M, int MH>
__global__ __launch_bounds__(256) void kv_write_kernel(KvGeom g, KvOperand<const T> k, KvOperand<const T> v, int vec) {
    constexpr int P = RowLanes<NB>::P, RB = 4 * NB * BITS;
    const int kv = blockIdx.y;
    const KvOperand<const T>& o = kv ? v : k;
    const int p = threadIdx.x % P;
    for (int i = blockIdx.z; i < g.n; i += gridDim.z) {
        const KvRow r = kv_row(g, i);
        typename KvEight<T>::v8 raw[M];                             // (turned into floats only when all are requested)
        int h[M], at[M];
        bool live[M];
#pragma unroll
        for (int m = 0; m < M; ++m) {
            const int unit = (blockIdx.x * (M / MH) + m / MH) * (256 / P) + (int)threadIdx.x / P, group = unit / g.T;
            const int t = unit - group * g.T;
            h[m] = group * MH + m % MH;
            at[m] = r.pos + t;
            live[m] = p < RowLanes<NB>::live && h[m] < g.H && r.e >= 0 && t < r.cnt && at[m] >= 0 && at[m] < g.S;
            raw[m] = (T)0.f;
            if (live[m]) kv_fetch8<T>(o.p + (long)i * o.row + (long)t * o.step + (long)h[m] * o.head + 8 * p, vec, raw[m]);
        }
        if (g.idx && r.e >= 0 && i + 1 < g.n) {                     // an episode listed twice: the last listing is the one that is written
            bool later = false;
            for (int j = i + 1 + (int)threadIdx.x; j < g.n; j += 256) later |= g.idx[j] == r.e;
            if (__syncthreads_or(later)) continue;
        }
#pragma unroll
        for (int m = 0; m < M; ++m) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = (float)raw[m][e];
            const unsigned sb = kv_scale_byte<BITS>(kv_block_top(x));
            unsigned w[BITS / 4];
            kv_encode8<BITS>(x, sb, w);
            unsigned word = sb;                                     // the row's scale bytes, gathered in its first lane
            if constexpr (NB >= 2) word |= __shfl_down(sb, 4, P) << 8;
            if constexpr (NB >= 3) word |= __shfl_down(sb, 8, P) << 16;
            if constexpr (NB >= 4) word |= __shfl_down(sb, 12, P) << 24;
            if (!live[m]) continue;
            unsigned char* c = g.codes + kv * g.ckv + (long)r.e * g.ce + (long)h[m] * g.ch + (long)at[m] * RB + p * BITS;
            if constexpr (BITS == 4) *(unsigned*)c = w[0];
            else *(uint2*)c = make_uint2(w[0], w[1]);
            if (p != 0) continue;
            unsigned char* sc = g.scales + kv * g.skv + (long)r.e * g.se + (long)h[m] * g.sh + (long)at[m] * 4;
            if constexpr (NB == 1) *sc = (unsigned char)word;
            else if constexpr (NB == 4) *(unsigned*)sc = word;
            else {
                *(unsigned short*)sc = (unsigned short)word;
                if constexpr (NB == 3) sc[2] = (unsigned char)(word >> 16);
            }
        }
    }
}

// eight codes -> numbers; the first and the last four with a scale of their own
template <int BITS> __device__ __forceinline__ void kv_decode8(const unsigned (&w)[BITS / 4], const unsigned (&scale_byte)[2], float (&x)[8]) {
    const float s0 = __uint_as_float(scale_byte[0] << 23), s1 = __uint_as_float(scale_byte[1] << 23);
    f32x2 y[4];
    if constexpr (BITS == 4) {
        y[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[0], s0, 0);
        y[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[0], s0, 1);
        y[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[0], s1, 2);
        y[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[0], s1, 3);
    } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            y[2 * h] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w[h], h ? s1 : s0, false);
            y[2 * h + 1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w[h], h ? s1 : s0, true);
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = y[i >> 1][i & 1];
}

// `second`: where the last four of the eight go (4 = behind the first)
template <typename T> __device__ __forceinline__ void kv_store8(T* p, bool vec, const float (&x)[8], int second) {
    if constexpr (sizeof(T) == 4) {
        if (vec) {
            *(f32x4*)p = (f32x4){x[0], x[1], x[2], x[3]};
            *(f32x4*)(p + second) = (f32x4){x[4], x[5], x[6], x[7]};
            return;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) p[(i & 4 ? second - 4 : 0) + i] = x[i];
    } else {
        typename Half16<T>::v8 o;
#pragma unroll
        for (int i = 0; i < 8; ++i)                                // exact in bf16; fp16: rounded below 2^-14
            o[i] = kv_result<T>(x[i]);
        if (vec) { *(typename Half16<T>::v8*)p = o; return; }
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = o[i];
    }
}

// A lane's eight numbers are neighbours in 16 bits; in fp32 it takes four of the row's first half and four of its second, so that each
// of its two 16-byte stores fills whole lines with its neighbours' (64 x 1500 steps x 6 heads of 64, 4 bits -> fp32 78 us against 91).
template <int NB, int BITS, typename T, int M, int MH>
__global__ __launch_bounds__(256) void kv_read_kernel(KvGeom g, KvOperand<T> k, KvOperand<T> v, int vec) {
    constexpr int P = RowLanes<NB>::P, RB = 4 * NB * BITS, NUM = sizeof(T) == 4 ? 4 : 8, HALF = sizeof(T) == 4 ? 16 * NB : 4;
    const int kv = blockIdx.y;
    const KvOperand<T>& o = kv ? v : k;
    const int p = threadIdx.x % P;
    if (p >= RowLanes<NB>::live) return;
    for (int i = blockIdx.z; i < g.n; i += gridDim.z) {
        const KvRow r = kv_row(g, i);
        unsigned w[M][BITS / 4], sb[M][2];
        int h[M], t[M];
#pragma unroll
        for (int m = 0; m < M; ++m) {
            const int unit = (blockIdx.x * (M / MH) + m / MH) * (256 / P) + (int)threadIdx.x / P, group = unit / g.T;
            t[m] = unit - group * g.T;
            h[m] = group * MH + m % MH;
            const int at = r.pos + t[m];
            sb[m][0] = sb[m][1] = 0;
#pragma unroll
            for (int q = 0; q < BITS / 4; ++q) w[m][q] = 0;
            if (h[m] < g.H && r.e >= 0 && t[m] < r.cnt && at >= 0 && at < g.S) {
                const unsigned char* c = g.codes + kv * g.ckv + (long)r.e * g.ce + (long)h[m] * g.ch + (long)at * RB + p * (NUM * BITS / 8);
                const unsigned char* sc = g.scales + kv * g.skv + (long)r.e * g.se + (long)h[m] * g.sh + (long)at * 4;
                sb[m][0] = sc[p * NUM / 32];
                if constexpr (NUM == 4) {
                    sb[m][1] = sc[(HALF + p * 4) / 32];
                    if constexpr (BITS == 4) w[m][0] = *(const unsigned short*)c | (unsigned)*(const unsigned short*)(c + RB / 2) << 16;
                    else { w[m][0] = *(const unsigned*)c; w[m][1] = *(const unsigned*)(c + RB / 2); }
                } else if constexpr (BITS == 4) {
                    w[m][0] = *(const unsigned*)c;
                } else {
                    const uint2 u = *(const uint2*)c;
                    w[m][0] = u.x; w[m][1] = u.y;
                }
            }
        }
#pragma unroll
        for (int m = 0; m < M; ++m) {
            if (h[m] >= g.H) continue;
            float x[8];
            if constexpr (NUM == 8) sb[m][1] = sb[m][0];
            kv_decode8<BITS>(w[m], sb[m], x);                       // (what does not exist: codes 0, the number 0)
            kv_store8<T>(o.p + (long)i * o.row + (long)t[m] * o.step + (long)h[m] * o.head + NUM * p, vec, x, HALF);
        }
    }
}

inline bool operand_vec(const otter_kv_operand* o, int dtype) {
    const long es = dtype == DT_F32 ? 4 : 2;
    return aligned16(o->p) && (o->row * es) % 16 == 0 && (o->step * es) % 16 == 0 && (o->head * es) % 16 == 0;
}

template <bool WRITE, int NB, int BITS, typename T, int M, int MH>
void launch_m(const KvGeom& g, const otter_kv_operand* k, const otter_kv_operand* v, int vec, hipStream_t s) {
    const long rows = (long)(g.H / MH) * g.T, a_block = M / MH * (256 / RowLanes<NB>::P);
    const dim3 grid((unsigned)((rows + a_block - 1) / a_block), 2, (unsigned)std::min(g.n, 65535));
    if constexpr (WRITE)
        hipLaunchKernelGGL((kv_write_kernel<NB, BITS, T, M, MH>), grid, dim3(256), 0, s, g, (KvOperand<const T>{(const T*)k->p, k->row, k->step, k->head}),
                           (KvOperand<const T>{(const T*)v->p, v->row, v->step, v->head}), vec);
    else
        hipLaunchKernelGGL((kv_read_kernel<NB, BITS, T, M, MH>), grid, dim3(256), 0, s, g, (KvOperand<T>{(T*)k->p, k->row, k->step, k->head}),
                           (KvOperand<T>{(T*)v->p, v->row, v->step, v->head}), vec);
}

// One piece a lane while that leaves the chip short of workgroups, four otherwise.  A wave that writes takes the same four rows of
// four heads where the heads allow: it reads runs of four heads (one projection's output holds q | k | v of a step, so a head alone
// is 256 bytes of 6 KB): 16 histories of 4093 steps x 8 heads of 128, bf16 -> 4 bits 72 us against 86 with sixteen rows of one head (other numbers
// each time).  Reading is as fast or faster along one head (56 us against 60).
template <bool WRITE, int NB, int BITS, typename T>
void launch(const KvGeom& g, const otter_kv_operand* k, const otter_kv_operand* v, int vec, hipStream_t s) {
    if ((long)g.H * g.T * RowLanes<NB>::P / 1024 * 2 * g.n >= 2048) {
        if (WRITE && g.H % 4 == 0) launch_m<WRITE, NB, BITS, T, 4, WRITE ? 4 : 1>(g, k, v, vec, s);
        else launch_m<WRITE, NB, BITS, T, 4, 1>(g, k, v, vec, s);
    } else {
        launch_m<WRITE, NB, BITS, T, 1, 1>(g, k, v, vec, s);
    }
}

template <bool WRITE, int BITS, typename T>
void launch_nb(int nb, const KvGeom& g, const otter_kv_operand* k, const otter_kv_operand* v, int vec, hipStream_t s) {
    if (nb == 1) launch<WRITE, 1, BITS, T>(g, k, v, vec, s);
    else if (nb == 2) launch<WRITE, 2, BITS, T>(g, k, v, vec, s);
    else if (nb == 3) launch<WRITE, 3, BITS, T>(g, k, v, vec, s);
    else launch<WRITE, 4, BITS, T>(g, k, v, vec, s);
}

template <bool WRITE>
int move(const otter_kv_cache* c, const otter_kv_rows* r, int dtype, const otter_kv_operand* k, const otter_kv_operand* v, hipStream_t s, const char* name) {
    if (int rc = otter_kv_check(c, r, name)) return rc;
    if (r->n_rows == 0 || r->steps == 0) return OTTER_OK;
    if (int rc = otter_kv_check_operand(k, dtype, !WRITE, "k", name)) return rc;
    if (int rc = otter_kv_check_operand(v, dtype, !WRITE, "v", name)) return rc;
    OTTER_REQUIRE((long)c->heads * r->steps * 16 < (1L << 31) - 1024, OTTER_ERR_UNSUPPORTED_SHAPE, "%s: %d heads x %d steps too large", name, c->heads, r->steps);
    if (WRITE)
        if (int rc = otter_kv_check_writable(c, name)) return rc;
    const KvGeom g = otter_kv_geom(c, r);
    const int vec = operand_vec(k, dtype) && operand_vec(v, dtype), nb = c->head_dim / 32;
    if (c->bits == 4) {
        if (dtype == DT_F32) launch_nb<WRITE, 4, float>(nb, g, k, v, vec, s);
        else if (dtype == DT_BF16) launch_nb<WRITE, 4, __bf16>(nb, g, k, v, vec, s);
        else launch_nb<WRITE, 4, _Float16>(nb, g, k, v, vec, s);
    } else {
        if (dtype == DT_F32) launch_nb<WRITE, 8, float>(nb, g, k, v, vec, s);
        else if (dtype == DT_BF16) launch_nb<WRITE, 8, __bf16>(nb, g, k, v, vec, s);
        else launch_nb<WRITE, 8, _Float16>(nb, g, k, v, vec, s);
    }
    OTTER_CHECK_LAUNCH(name);
    return OTTER_OK;
}

}  // namespace

int otter_kv_check(const otter_kv_cache* c, const otter_kv_rows* r, const char* name) {
    OTTER_REQUIRE(c && r && c->codes && c->scales, OTTER_ERR_INVALID_ARGUMENT, "%s: null cache", name);
    OTTER_REQUIRE(c->bits == 4 || c->bits == 8, OTTER_ERR_INVALID_ARGUMENT, "%s: %d bits (4 or 8)", name, c->bits);
    OTTER_REQUIRE(c->head_dim >= 32 && c->head_dim <= 128 && c->head_dim % 32 == 0, OTTER_ERR_UNSUPPORTED_SHAPE,
                  "%s: head_dim=%d must be 32, 64, 96 or 128", name, c->head_dim);
    OTTER_REQUIRE(c->episodes >= 0 && c->heads > 0 && c->capacity > 0 && c->capacity <= (1 << 30), OTTER_ERR_INVALID_ARGUMENT,
                  "%s: episodes=%d heads=%d capacity=%d", name, c->episodes, c->heads, c->capacity);
    const long row = (long)c->head_dim * c->bits / 8;
    OTTER_REQUIRE(aligned16(c->codes) && c->code_kv % 16 == 0 && c->code_episode % 16 == 0 && c->code_head % 16 == 0, OTTER_ERR_ALIGNMENT,
                  "%s: codes and their strides must be multiples of 16 bytes", name);
    OTTER_REQUIRE((reinterpret_cast<uintptr_t>(c->scales) & 3u) == 0 && c->scale_kv % 4 == 0 && c->scale_episode % 4 == 0 && c->scale_head % 4 == 0,
                  OTTER_ERR_ALIGNMENT, "%s: scales and their strides must be multiples of 4 bytes", name);
    OTTER_REQUIRE((c->heads == 1 || c->code_head >= c->capacity * row) && (c->heads == 1 || c->scale_head >= c->capacity * 4L),
                  OTTER_ERR_INVALID_ARGUMENT, "%s: heads of the cache overlap", name);
    OTTER_REQUIRE(r->n_rows >= 0 && r->steps >= 0 && r->steps <= (1 << 30), OTTER_ERR_INVALID_ARGUMENT, "%s: n_rows=%d steps=%d", name, r->n_rows, r->steps);
    OTTER_REQUIRE(r->idx || r->n_rows <= c->episodes, OTTER_ERR_INVALID_ARGUMENT, "%s: %d rows without idx, cache of %d episodes", name, r->n_rows, c->episodes);
    return OTTER_OK;
}

// (reading, episodes may share rows; what is written has rows of its own)
int otter_kv_check_writable(const otter_kv_cache* c, const char* name) {
    const long row = (long)c->head_dim * c->bits / 8;
    OTTER_REQUIRE((c->episodes <= 1 || (c->code_episode >= c->capacity * row && c->scale_episode >= c->capacity * 4L)) &&
                      c->code_kv >= c->capacity * row && c->scale_kv >= c->capacity * 4L,
                  OTTER_ERR_INVALID_ARGUMENT, "%s: episodes, or keys and values, of the cache overlap", name);
    return OTTER_OK;
}

int otter_kv_check_operand(const otter_kv_operand* o, int dtype, bool write, const char* what, const char* name) {
    OTTER_REQUIRE(dtype == DT_BF16 || dtype == DT_F16 || dtype == DT_F32, OTTER_ERR_INVALID_ARGUMENT, "%s: unknown dtype %d", name, dtype);
    OTTER_REQUIRE(o && o->p, OTTER_ERR_INVALID_ARGUMENT, "%s: null operand %s", name, what);
    OTTER_REQUIRE((reinterpret_cast<uintptr_t>(o->p) & (dtype == DT_F32 ? 3u : 1u)) == 0, OTTER_ERR_ALIGNMENT, "%s: %s is not aligned to its elements", name, what);
    OTTER_REQUIRE(!write || (o->row >= 0 && o->step >= 0 && o->head >= 0), OTTER_ERR_INVALID_ARGUMENT, "%s: negative strides of %s", name, what);
    return OTTER_OK;
}

KvGeom otter_kv_geom(const otter_kv_cache* c, const otter_kv_rows* r) {
    return KvGeom{c->codes, c->code_kv, c->code_episode, c->code_head, c->scales, c->scale_kv, c->scale_episode, c->scale_head,
                  c->episodes, c->capacity, c->heads, r->idx, r->pos, r->count, r->n_rows, r->steps};
}

extern "C" int otter_kv_cache_write(const otter_kv_cache* cache, const otter_kv_rows* rows, int dtype, const otter_kv_operand* k,
                                    const otter_kv_operand* v, void* stream) {
    return move<true>(cache, rows, dtype, k, v, (hipStream_t)stream, "otter_kv_cache_write");
}

extern "C" int otter_kv_cache_read(const otter_kv_cache* cache, const otter_kv_rows* rows, int dtype, const otter_kv_operand* k,
                                   const otter_kv_operand* v, void* stream) {
    return move<false>(cache, rows, dtype, k, v, (hipStream_t)stream, "otter_kv_cache_read");
}
