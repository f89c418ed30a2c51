"""The quantised K/V cache without a GPU: the plain implementation that the GPU tests compare with, the operators' registration
and shapes, and every refusal of the C entry points (all of them come before anything is launched)."""
import ctypes
import math

import pytest
import torch

import kv_plain as P
from otter_amd import _lib

ADDR = 1 << 20                                          # never dereferenced: every call below is refused or has no rows


# ---------------------------------------------------------------------------------------------------- the plain implementation
def test_plain_e4m3_agrees_with_torch():
    x = torch.randn(40, 128, generator=torch.Generator().manual_seed(0)) * torch.logspace(-6, 6, 40)[:, None]
    codes, scales = P.quantise(x, 8)
    e = scales[:, :4].double().repeat_interleave(32, -1) - 127
    want = (x.double() * 2.0 ** -e).clamp(-448, 448).to(torch.float8_e4m3fn)
    assert torch.equal(codes, want.view(torch.uint8))
    assert torch.equal(P.dequantise(codes, scales, 8), want.double() * 2.0 ** e)
    top = x.abs().view(40, 4, 32).amax(-1).double()
    s = 2.0 ** (scales[:, :4].double() - 127)
    assert bool((top <= 448 * s).all()) and bool((top > 224 * s).all())


def test_plain_e2m1_by_hand():
    x = torch.zeros(1, 32)
    x[0, :13] = torch.tensor([6.0, 0.25, 0.26, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 5.01, -0.25, -2.5, -6.0])
    codes, scales = P.quantise(x, 4)
    assert int(scales[0, 0]) == 127
    got = P.dequantise(codes, scales, 4)[0, :13]
    assert torch.equal(got, torch.tensor([6, 0, 0.5, 1, 1, 2, 2, 4, 4, 6, 0, -2, -6], dtype=torch.float64))
    assert int(codes[0, 0]) == 7 | (0 << 4) and int(codes[0, 1]) == 1 | (2 << 4)          # the even number in the low half
    y = torch.full((1, 32), 6.001)
    assert int(P.quantise(y, 4)[1][0, 0]) == 128
    z = torch.zeros(1, 32)
    z[0, 3] = math.nan
    c, s = P.quantise(z, 4)
    assert int(s[0, 0]) == 255 and bool(torch.isnan(P.dequantise(c, s, 4)).all())


# ---------------------------------------------------------------------------------------------------- operators
def test_operators_are_registered_with_shapes_and_no_cpu_implementation():
    import otter_amd.kv_cache as K
    ns = torch.ops.otter_hip
    assert K.OP_NAMES == ("kv_cache_write", "kv_cache_read", "attn_cache", "attn_cache_rows")
    meta = lambda *s, dtype=torch.bfloat16: torch.empty(*s, dtype=dtype, device="meta")          # noqa: E731
    codes, scales = meta(2, 5, 2, 40, 48, dtype=torch.uint8), meta(2, 5, 2, 40, 4, dtype=torch.uint8)
    i32 = meta(3, dtype=torch.int32)
    assert ns.kv_cache_write(meta(3, 7, 2, 96), meta(3, 7, 2, 96), codes, scales, None, i32, None) is None
    k, v = ns.kv_cache_read(codes, scales, 96, 7, None, i32, None, -1, 1)
    assert tuple(k.shape) == tuple(v.shape) == (3, 7, 2, 96) and k.dtype == torch.float16
    assert tuple(ns.kv_cache_read(codes, scales, 96, 7, None, None, None, -1, 2)[0].shape) == (5, 7, 2, 96)
    y = ns.attn_cache(meta(3, 7, 4, 96), codes, scales, None, i32, None, True, 0, None, None)
    assert tuple(y.shape) == (3, 7, 4, 96) and y.dtype == torch.bfloat16
    assert tuple(ns.attn_cache_rows(meta(3, 4, 96), meta(3, 2, 96), meta(3, 2, 96), codes, scales, None, i32, 0, None, None).shape) == (3, 4, 96)
    c = K.KVCache(1, 1, 4, 32, 4, "cpu")
    assert (c.episodes, c.heads, c.capacity, c.nbytes) == (1, 1, 4, 2 * 4 * (16 + 4))
    x = torch.zeros(1, 1, 1, 32)
    for call in (lambda: c.write(x, x), lambda: c.read(1), lambda: c.attend(x), lambda: c.step(x[0], x[0], x[0])):
        with pytest.raises(NotImplementedError):
            call()


@pytest.mark.parametrize("args", [dict(bits=3), dict(head_dim=48), dict(head_dim=160), dict(head_dim=0), dict(heads=0), dict(capacity=0)])
def test_cache_refuses(args):
    from otter_amd.kv_cache import KVCache
    with pytest.raises(ValueError):
        KVCache(**{**dict(episodes=1, heads=1, capacity=4, head_dim=32, bits=4, device="cpu"), **args})


def test_wrappers_refuse_host_tensors():
    from otter_amd import ops
    codes, scales = torch.zeros(2, 1, 1, 4, 16, dtype=torch.uint8), torch.zeros(2, 1, 1, 4, 4, dtype=torch.uint8)
    x = torch.zeros(1, 1, 1, 32)
    for call in (lambda: ops.kv_cache_write(x, x, codes, scales), lambda: ops.kv_cache_read(codes, scales, 32, 1), lambda: ops.attn_cache(x, codes, scales),
                 lambda: ops.attn_cache_rows(x[0], x[0], x[0], codes, scales)):
        with pytest.raises(ops.OtterHipError):
            call()
    with pytest.raises(ValueError):
        ops.attn_cache(x[0], codes, scales)
    with pytest.raises(ValueError):
        ops.kv_cache_write(x[0], x[0], codes, scales)
    with pytest.raises(ValueError):
        ops.attn_cache_rows(x, x, x, codes, scales)


# ---------------------------------------------------------------------------------------------------- C entry points
def _cache(**kw):
    f = dict(codes=ADDR, code_kv=1 << 16, code_episode=1 << 12, code_head=1 << 10, scales=ADDR, scale_kv=1 << 12, scale_episode=1 << 10,
             scale_head=1 << 8, bits=4, episodes=4, heads=2, capacity=16, head_dim=64)
    f.update(kw)
    return _lib.KvCache(**f)


def _rows(**kw):
    f = dict(idx=None, pos=None, count=None, n_rows=2, steps=1)
    f.update(kw)
    return _lib.KvRows(**f)


def _operand(**kw):
    f = dict(p=ADDR, row=256, step=128, head=64)
    f.update(kw)
    return _lib.KvOperand(**f)


BAD_CACHES = [dict(bits=5), dict(head_dim=48), dict(head_dim=256), dict(head_dim=0), dict(codes=None), dict(scales=None), dict(codes=ADDR + 8), dict(scales=ADDR + 2),
              dict(code_head=1000), dict(scale_head=66), dict(code_head=16 * 32 - 16), dict(scale_head=60), dict(capacity=0), dict(heads=0), dict(episodes=-1)]
BAD_ROWS = [dict(n_rows=-1), dict(steps=-1), dict(n_rows=5)]


def _refused(rc, *words):
    assert rc != 0
    msg = _lib.load().otter_last_error().decode()
    assert msg and all(w in msg for w in words), msg
    return msg


@pytest.mark.parametrize("entry", ["otter_kv_cache_write", "otter_kv_cache_read"])
def test_write_and_read_refuse(entry):
    fn = getattr(_lib.load(), entry)
    for bad in BAD_CACHES:
        _refused(fn(_cache(**bad), _rows(), 2, _operand(), _operand(), None), entry)
    for bad in BAD_ROWS:
        _refused(fn(_cache(), _rows(**bad), 2, _operand(), _operand(), None), entry)
    _refused(fn(_cache(), _rows(), 3, _operand(), _operand(), None), "dtype")
    for bad in (dict(p=None), dict(p=ADDR + 1)):
        _refused(fn(_cache(), _rows(), 2, _operand(**bad), _operand(), None), "k")
        _refused(fn(_cache(), _rows(), 1, _operand(), _operand(**bad), None), "v")
    _refused(fn(_cache(heads=1, capacity=1 << 20), _rows(steps=1 << 28), 2, _operand(), _operand(), None), "too large")
    assert fn(_cache(), _rows(n_rows=0), 2, None, None, None) == 0                       # nothing to do
    assert fn(_cache(), _rows(steps=0), 2, None, None, None) == 0


def test_attention_refuses():
    lib = _lib.load()
    fn = lib.otter_attn_cache

    def call(cache=None, rows=None, dtype=2, q=None, heads=2, k=None, v=None, out=None, causal=1, window=0, max_len=16, scale=0.1, ws=None, n_ws=0):
        return fn(cache or _cache(), rows or _rows(), dtype, q or _operand(), heads, k, v, out or _operand(), causal, window, max_len, scale, ws, n_ws, None)

    for bad in BAD_CACHES:
        _refused(call(cache=_cache(**bad)), "otter_attn_cache")
    for bad in BAD_ROWS:
        _refused(call(rows=_rows(**bad)), "otter_attn_cache")
    _refused(call(cache=_cache(episodes=0), rows=_rows(n_rows=0)) or call(cache=_cache(episodes=0), rows=_rows(idx=ADDR)), "no episodes")
    for h in (0, -2, 3):
        _refused(call(heads=h), "query heads")
    for kw in (dict(window=-1), dict(max_len=0), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf)):
        _refused(call(**kw))
    _refused(call(dtype=7), "dtype")
    _refused(call(q=_operand(p=None)), "q")
    for bad in (dict(p=ADDR + 4), dict(row=250), dict(head=66), dict(row=-256)):
        _refused(call(out=_operand(**bad)), "out")
    _refused(call(k=_operand()), "together")
    _refused(call(rows=_rows(steps=2), k=_operand(), v=_operand()), "one step")
    _refused(call(rows=_rows(count=ADDR), k=_operand(), v=_operand()), "one step")
    # a split launch without (enough, aligned) scratch
    big = _cache(capacity=8192, code_head=1 << 20, code_episode=1 << 21, code_kv=1 << 24, scale_head=1 << 15, scale_episode=1 << 16, scale_kv=1 << 20)
    need = lib.otter_attn_cache_workspace_floats(2, 2, 1, 2, 2, 64, 0, 8192)
    assert need > 0
    _refused(call(cache=big, max_len=8192), "workspace")
    _refused(call(cache=big, max_len=8192, ws=ADDR, n_ws=need - 1), "workspace")
    _refused(call(cache=big, max_len=8192, ws=ADDR + 4, n_ws=need), "workspace")
    assert lib.otter_attn_cache_workspace_floats(2, 2, 1, 2, 2, 64, 0, 32) == 0           # short histories need none
    for bad in ((2, 0, 1, 2, 2, 64, 0, 64), (2, 1, 1, 3, 2, 64, 0, 64), (2, 1, 1, 2, 2, 64, 0, 0), (2, 1, 1, 2, 2, 64, -1, 64), (2, 1 << 30, 1 << 30, 2, 2, 64, 0, 64)):
        assert lib.otter_attn_cache_workspace_floats(*bad) == 0
    assert call(rows=_rows(n_rows=0)) == 0 and call(rows=_rows(steps=0)) == 0


def test_workspace_covers_every_plan():
    """The scratch that the sizing function names is what the launch asks for, over the plans' whole range (the refusal names it)."""
    lib = _lib.load()
    import random
    rng = random.Random(3)
    split = 0
    for _ in range(300):
        dtype, d, h = rng.choice([0, 1, 2]), rng.choice([32, 64, 96, 128]), rng.choice([1, 2, 8])
        hq, n, steps = h * rng.choice([1, 3, 8, 40]), rng.choice([1, 2, 33, 600]), rng.choice([1, 2, 17, 300])
        cap, window = rng.choice([31, 100, 1000, 9000]), rng.choice([0, 0, 64, 5000])
        need = lib.otter_attn_cache_workspace_floats(dtype, n, steps, hq, h, d, window, cap)
        if not need:
            continue
        split += 1
        row = d // 2
        cache = _cache(head_dim=d, heads=h, episodes=n, capacity=cap, code_head=cap * row, code_episode=h * cap * row, code_kv=n * h * cap * row,
                       scale_head=cap * 4, scale_episode=h * cap * 4, scale_kv=n * h * cap * 4)
        op = _operand(row=steps * hq * d, step=hq * d, head=d)
        rc = lib.otter_attn_cache(cache, _rows(n_rows=n, steps=steps), dtype, op, hq, None, None, op, 1, window, cap, 0.1, ADDR, need - 1, None)
        _refused(rc, f"workspace of {need} floats")
    assert split > 50


def test_overlapping_episodes_are_not_written():
    """Episodes that share rows (an expanded cache) can be read and attended to, never written."""
    lib = _lib.load()
    for bad in (dict(code_episode=0), dict(scale_episode=0), dict(code_kv=0), dict(scale_kv=0), dict(code_episode=16 * 32 - 16)):
        _refused(lib.otter_kv_cache_write(_cache(**bad), _rows(), 2, _operand(), _operand(), None), "overlap")
        _refused(lib.otter_attn_cache(_cache(**bad), _rows(), 2, _operand(), 2, _operand(), _operand(), _operand(), 1, 0, 16, 0.1, None, 0, None), "overlap")


def test_attention_refuses_what_no_launch_holds():
    lib = _lib.load()
    for scale in (1.0e38, 3.0e38):                                                       # scale log2(e) would leave fp32
        _refused(lib.otter_attn_cache(_cache(), _rows(), 2, _operand(), 2, None, None, _operand(), 1, 0, 16, scale, None, 0, None), "scale")
    # 2^26 rows of one head: one workgroup takes four, a grid has 2^32 threads
    many = _cache(heads=1, episodes=1 << 27)
    _refused(lib.otter_attn_cache(many, _rows(n_rows=1 << 27), 2, _operand(), 1, None, None, _operand(), 1, 0, 16, 0.1, None, 0, None), "grid")


def test_the_compiled_way_leaves_what_it_does_not_take():
    """Anything but whole device tensors of the right kind: None, nothing done, nothing raised."""
    b = _lib.kv_binding()
    codes, scales = torch.zeros(2, 1, 1, 4, 16, dtype=torch.uint8), torch.zeros(2, 1, 1, 4, 4, dtype=torch.uint8)
    x = torch.zeros(1, 1, 1, 32)
    sparse = torch.zeros(1, 1, 1, 32).to_sparse()
    for k in (x, x[0], sparse, None, 3, "k", torch.zeros(1, 1, 1, 32, device="meta"), torch.nn.Parameter(x)):
        for c, s in ((codes, scales), (scales, codes), (None, scales), (codes, sparse), (sparse, sparse), (codes.to("meta"), scales.to("meta"))):
            assert b.write(k, k, c, s, None, None, None) is None
            assert b.attend(k, None, None, c, s, None, None, None, True, 0, None, None) is None
            assert b.attend(k, k, k, c, s, None, None, None, True, 0, None, None) is None
            assert b.read(c, s, 32, 1, None, None, None, None, 2) is None
    assert b.write() is None and b.read(codes) is None and b.attend(x, x) is None
    assert b.read(codes, scales, "32", 1, None, None, None, None, 2) is None and b.read(codes, scales, 1 << 70, 1, None, None, None, None, 2) is None
