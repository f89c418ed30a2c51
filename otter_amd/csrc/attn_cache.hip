// Entry points of the attention over the quantised cache: argument checks and how the work is dealt out (kernel: attn_cache.hpp).
#include <algorithm>

#include "attn_cache.hpp"

namespace {

struct Plan { int qt, vec, wide, cg, kw, nsplit, chunk; unsigned blocks; bool ok; };

inline long ceil_div(long a, long b) { return (a + b - 1) / b; }

// Into how many splits the keys of each of `items` workgroups' worth of work are cut.  A compute unit holds R workgroups at a time, and
// R of them together take R units of time; k < R of them are slower than that (a unit has nothing else to do while they wait for
// memory), a lone one by `lone`.  Every split of the keys costs `join` of an item (its prologue, its sums written and read again).
// Measured (one position, 32 / 8 heads of 128, 8000 keys in 4 bits; items: us at 1, 2, 3, 4 splits): 256: 95 67 61 71; 320: 108 77 87 78;
// 384: 111 85 95 88; 480: 115 126 110 113.  At 640 items of 1000 keys one split takes 21 us, two 26.
int splits(long items, int R, double lone, double join, long most) {
    constexpr long units = 256;
    if (items >= R * units) return 1;
    int best = 1;
    double least = 1e30;
    for (long ns = 1; ns <= std::min<long>(most, 128); ++ns) {
        const long m = ceil_div(items * ns, units), k = m % R;
        const double time = ((m - k) + (k ? k + lone * (1.0 - (double)(k - 1) / (R - 1)) : 0.0)) / ns + (ns > 1 ? ns * join * items / units : 0.0);
        if (time < least) { least = time; best = (int)ns; }
    }
    return best;
}

// One step with one or two query heads a key head: the vector form.  Columns otherwise: 16 per wave while all of a row's columns fit,
// then 32; from 33 on, with several steps, four waves share the converted tiles.
// Keys: one wave (wide: one workgroup) walks over all of them while there are enough to fill the chip, four waves and several
// workgroups share them otherwise.
Plan plan(int dtype, int nb, int n, int H, int steps, int G, int window, int max_len) {
    Plan p{};
    const long U = (long)n * H, N = (long)steps * G;
    p.vec = steps == 1 && G <= 2;
    p.wide = N > 32 && steps > 1;
    // (narrow: 32 only where that leaves two waves a SIMD: few waves are a matter of latency, not of conversions)
    p.qt = N <= 16 || (p.wide ? N <= 64 || wide_columns(dtype, nb) == 1 : U * ceil_div(N, 32) < 2048 || narrow_columns(dtype, nb) == 1) ? 1 : 2;
    const long cols = (p.wide ? 64L : 16L) * p.qt;
    p.cg = (int)ceil_div(N, cols);
    const long span = (window > 0 ? std::min<long>(max_len, (long)window + cols / G + 1) : max_len) + 31;   // keys one item may walk over
    const long items = U * p.cg;
    p.kw = (!p.wide && span > 95 && items < 4096) ? 4 : 1;
    p.nsplit = 1;
    p.chunk = (int)(ceil_div(span, 128) * 128);
    if (p.kw == 4 || p.wide) {
        // (registers decide how many workgroups a unit holds: the kernels' launch bounds)
        const int R = p.vec ? (G == 1 ? 4 : 3) : p.wide ? (nb <= 2 ? 3 : 2) : narrow_groups(dtype, nb, p.qt);
        const double keys = (double)std::max(span - steps / 2, 1L);                                  // about what the steps see of a causal span
        const int ns = splits(items, R, p.wide ? 0.35 : 0.75, (p.wide ? 400.0 : 300.0) / keys, ceil_div(span, p.wide ? 512 : 256));
        p.chunk = (int)(ceil_div(ceil_div(span, ns), 128) * 128);
        p.nsplit = (int)ceil_div(span, p.chunk);
    }
    const long blocks = p.wide || p.kw == 4 ? items * p.nsplit : p.cg == 1 ? ceil_div(U, 4) : U * ceil_div(p.cg, 4);
    p.ok = blocks < (1L << 24);                                     // (a grid has at most 2^32 threads a dimension)
    p.blocks = (unsigned)blocks;
    return p;
}

}  // namespace

extern "C" long otter_attn_cache_workspace_floats(int dtype, int n_rows, int steps, int q_heads, int kv_heads, int head_dim, int window, int max_len) {
    if (n_rows <= 0 || steps <= 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads != 0 || head_dim <= 0 || max_len <= 0 || window < 0) return 0;
    if ((long)steps * (q_heads / kv_heads) >= (1L << 31) || (long)n_rows * kv_heads >= (1L << 31)) return 0;
    const Plan p = plan(dtype, head_dim / 32, n_rows, kv_heads, steps, q_heads / kv_heads, window, max_len);
    return p.nsplit > 1 ? (long)p.nsplit * n_rows * q_heads * steps * (head_dim + 2) : 0;
}

extern "C" int otter_attn_cache(const otter_kv_cache* cache, const otter_kv_rows* rows, int dtype, const otter_kv_operand* q, int q_heads,
                                const otter_kv_operand* k_new, const otter_kv_operand* v_new, const otter_kv_operand* out, int causal,
                                int window, int max_len, float scale, float* workspace, long workspace_floats, void* stream) {
    const char* name = "otter_attn_cache";
    if (int rc = otter_kv_check(cache, rows, name)) return rc;
    if (rows->n_rows == 0 || rows->steps == 0) return OTTER_OK;
    OTTER_REQUIRE(cache->episodes > 0, OTTER_ERR_INVALID_ARGUMENT, "%s: the cache has no episodes", name);
    OTTER_REQUIRE(q_heads > 0 && q_heads % cache->heads == 0, OTTER_ERR_UNSUPPORTED_SHAPE, "%s: %d query heads over %d key heads", name, q_heads, cache->heads);
    OTTER_REQUIRE(window >= 0 && max_len > 0, OTTER_ERR_INVALID_ARGUMENT, "%s: window=%d max_len=%d", name, window, max_len);
    OTTER_REQUIRE(scale > 0.f && scale < 1.0e38f, OTTER_ERR_INVALID_ARGUMENT, "%s: scale must be positive and finite", name);
    if (int rc = otter_kv_check_operand(q, dtype, false, "q", name)) return rc;
    if (int rc = otter_kv_check_operand(out, dtype, true, "out", name)) return rc;
    const long es = dtype == DT_F32 ? 4 : 2;
    auto vec = [es](const otter_kv_operand* o) { return aligned16(o->p) && (o->row * es) % 16 == 0 && (o->step * es) % 16 == 0 && (o->head * es) % 16 == 0; };
    OTTER_REQUIRE(vec(out), OTTER_ERR_ALIGNMENT, "%s: out and its strides must be multiples of 16 bytes", name);
    OTTER_REQUIRE((k_new == nullptr) == (v_new == nullptr), OTTER_ERR_INVALID_ARGUMENT, "%s: k_new and v_new come together", name);
    if (k_new) {
        OTTER_REQUIRE(rows->steps == 1 && !rows->count, OTTER_ERR_UNSUPPORTED_SHAPE, "%s: appends one step to every listed row (steps=%d, no count)", name, rows->steps);
        if (int rc = otter_kv_check_operand(k_new, dtype, false, "k_new", name)) return rc;
        if (int rc = otter_kv_check_operand(v_new, dtype, false, "v_new", name)) return rc;
        if (int rc = otter_kv_check_writable(cache, name)) return rc;
    }
    const int G = q_heads / cache->heads;
    OTTER_REQUIRE((long)rows->steps * G < (1L << 30) && (long)rows->n_rows * cache->heads < (1L << 30), OTTER_ERR_UNSUPPORTED_SHAPE, "%s: too many rows, heads or steps", name);
    const int cap = std::min(max_len, cache->capacity);
    Plan p = plan(dtype, cache->head_dim / 32, rows->n_rows, cache->heads, rows->steps, G, window, cap);
    OTTER_REQUIRE(p.ok, OTTER_ERR_UNSUPPORTED_SHAPE, "%s: grid too large", name);
    if (p.nsplit > 1) {
        const long need = (long)p.nsplit * rows->n_rows * q_heads * rows->steps * (cache->head_dim + 2);
        OTTER_REQUIRE(workspace && workspace_floats >= need && (reinterpret_cast<uintptr_t>(workspace) & 7u) == 0, OTTER_ERR_INVALID_ARGUMENT,
                      "%s: needs a workspace of %ld floats (8-byte aligned), got %ld", name, need, workspace ? workspace_floats : 0L);
    }
    AttnCacheArgs a{};
    a.g = otter_kv_geom(cache, rows);
    a.q = {q->p, q->row, q->step, q->head};
    a.q_vec = vec(q);
    a.out = {out->p, out->row, out->step, out->head};
    if (k_new) {
        a.kn = {k_new->p, k_new->row, 0, k_new->head};
        a.vn = {v_new->p, v_new->row, 0, v_new->head};
        a.new_vec = vec(k_new) && vec(v_new);
    }
    a.G = G;
    a.N = rows->steps * G;
    a.CG = p.cg;
    a.causal = causal ? 1 : 0;
    a.window = window;
    a.max_len = cap;
    a.c = scale * 1.44269504088896341f;
    a.vec = p.vec;
    a.wide = p.wide;
    a.longest = p.wide && p.nsplit == 1 && a.causal && window == 0 && rows->n_rows > 1 && rows->n_rows <= 64;
    a.kw = p.kw;
    a.nsplit = p.nsplit;
    a.chunk = p.chunk;
    a.part = workspace;
    const int nb = cache->head_dim / 32;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == DT_F32) return otter_attn_cache_launch<float>(a, nb, cache->bits, p.qt, p.blocks, s);
    if (dtype == DT_BF16) return otter_attn_cache_launch<__bf16>(a, nb, cache->bits, p.qt, p.blocks, s);
    return otter_attn_cache_launch<_Float16>(a, nb, cache->bits, p.qt, p.blocks, s);
}
