"""The rollout engine with a quantised K/V history: every mode of a step (cached, mixed, recompute: windows that slide), partial resets and sliding
windows, against the policy in 64 bits on the keys and values that the cache really holds."""
import numpy as np
import pytest
import torch

import golden_inputs as GI

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from otter_amd import _lib
    _lib.load()
    return torch.device("cuda:0")


def _model(dev, seq_length, seed, **kw):
    from otter_amd.config import ModelConfig, SharedConfig
    from otter_amd.otter import OTTER
    from otter_amd.params import otter_specs, random_state_dict
    mc = ModelConfig(**{**dict(clip_model="tiny-test", transformer_dim=128, transformer_layers=2, transformer_heads=2, vision_pooling_output_dim=128,
                               text_pooling_output_dim=64, proprio_hidden_dim=64, proprio_output_dim=32, pooling_heads=4), **kw})
    sc = SharedConfig(image_size=112, seq_length=seq_length, action_horizon=4)
    sd = random_state_dict(otter_specs(mc, sc), seed=seed)
    model = OTTER(mc, sc)
    model.load_state_dict(sd, strict=True)
    return model.to(dev).eval(), {k: v.double() for k, v in sd.items() if not k.startswith("clip_model.")}, mc


def _observations(steps, b, seed):
    rng = np.random.default_rng(seed)
    images = torch.from_numpy(rng.integers(0, 256, (steps, b, 2, 3, 112, 112), dtype=np.uint8))
    proprio = torch.from_numpy(rng.standard_normal((steps, b, 10)).astype(np.float32))
    return images, proprio, GI._tokens(rng, b, (4, 7, 9))


def _newest_action(ro, sd, e, heads):
    """The action chunk of episode e's newest position in 64 bits: window input and cached K/V from the engine, the rest from the
    weights; the cached K/V of that position are held to the format's half step."""
    import torch.nn.functional as F
    n = int(ro.lens_host[e])
    lin = lambda x, p: x @ sd[p + ".weight"].T + sd[p + ".bias"]                    # noqa: E731
    ln = lambda x, p: F.layer_norm(x, x.shape[-1:], sd[p + ".weight"], sd[p + ".bias"], 1e-5)   # noqa: E731
    x = ro.window[e, n - 1].double().cpu() + sd["pe.pe"][0, n - 1]
    dim = x.shape[0]
    hd = dim // heads
    idx = torch.tensor([e], dtype=torch.int32, device=ro.dev.device)
    for i, kv in enumerate(ro._cache):
        p = f"policy.layers.{i}."
        h = ln(x, p + "pre_ln")
        q, k, v = (lin(h, p + "attention." + nm).view(heads, hd) for nm in ("query", "key", "value"))
        kc, vc = (t[0].double().cpu() for t in kv.read(n, idx=idx))                  # (n, heads, hd)
        for got, want in ((kc[-1], k), (vc[-1], v)):
            top = want.view(heads, -1, 32).abs().amax(-1, keepdim=True).expand(-1, -1, 32).reshape(heads, hd)
            # 4 bits: half of the widest step, 2 * 2^e with 3 * 2^e < top; 8 bits: 2^-4 of the number or half the smallest step;
            # fp32 arithmetic in front of it adds 1e-4 of the block
            half = top / 3 if kv.bits == 4 else torch.maximum(want.abs() * 2.0 ** -4, top * 2.0 ** -17)
            assert bool(((got - want).abs() <= half * (1 + 1e-3) + 1e-4 * top).all())
        s = torch.einsum("hd,nhd->hn", q, kc) / hd ** 0.5
        a = torch.einsum("hn,nhd->hd", torch.softmax(s, -1), vc).reshape(dim)
        x = x + lin(a, p + "attention.out")
        h = ln(x, p + "post_ln")
        x = x + lin(F.gelu(lin(h, p + "mlp.0")), p + "mlp.2")
    return lin(torch.relu(lin(x, "action_head.mlp.0")), "action_head.mlp.2")


@pytest.mark.parametrize("bits", [4, 8])
def test_staggered_episodes_on_a_quantised_history(dev, bits):
    from otter_amd.engine import BatchedRollout
    model, sd, mc = _model(dev, 8, 41)
    d = model.device_model()
    B, steps = 5, 22
    resets = {2: [1], 3: [3, 4], 5: [0], 9: [2], 13: [1, 4], 17: [0, 1, 2, 3, 4], 19: [2]}
    images, proprio, text = _observations(steps, B, 19)
    tf = d.clip.text_tokens_cached(text)
    batch = BatchedRollout(d, B, kv_bits=bits)
    assert all(c.bits == bits for c in batch._cache)
    modes, worst = [], 0.0
    for t in range(steps):
        if t in resets:
            batch.reset(resets[t])
        got = batch.step(images[t].reshape(B * 2, 3, 112, 112).to(dev), tf, proprio[t].to(dev)).cpu().double()
        modes.append(batch.last_mode)
        for e in range(B):
            worst = max(worst, float((got[e].reshape(-1) - _newest_action(batch, sd, e, mc.transformer_heads)).abs().max()))
    print(f"{bits}-bit history: modes {''.join(m[0] for m in modes)}, max |action - 64 bits| = {worst:.2e}")
    assert {"cached", "mixed"} <= set(modes) and worst <= 1e-4           # the fp32 path's own tolerance


def test_window_past_64_positions(dev):
    """A window that the fp32 history cannot hold: filled step by step, then sliding (whole windows of 72 again every step)."""
    from otter_amd.engine import BatchedRollout
    model, sd, mc = _model(dev, 72, 43, transformer_dim=192, transformer_layers=1)    # head width 96
    d = model.device_model()
    B, steps = 2, 75
    images, proprio, text = _observations(steps, B, 23)
    tf = d.clip.text_tokens_cached(text)
    batch = BatchedRollout(d, B, kv_bits=4)
    for t in range(steps):
        got = batch.step(images[t].reshape(B * 2, 3, 112, 112).to(dev), tf, proprio[t].to(dev)).cpu().double()
        assert batch.last_mode == ("cached" if t < 72 else "recompute")
        if t in (0, 1, 40, 70, 71, 72, 74):
            for e in range(B):
                assert float((got[e].reshape(-1) - _newest_action(batch, sd, e, mc.transformer_heads)).abs().max()) <= 1e-4


def test_adopted_episodes_fill_their_rows_again(dev):
    """Windows handed over without K/V: the recompute step writes the episodes' own rows, after which they are cached again."""
    from otter_amd.engine import BatchedRollout
    model, sd, mc = _model(dev, 8, 47)
    d = model.device_model()
    B = 3
    images, proprio, text = _observations(6, B, 29)
    tf = d.clip.text_tokens_cached(text)
    first = BatchedRollout(d, B, kv_bits=8)
    for t in range(3):
        first.step(images[t].reshape(B * 2, 3, 112, 112).to(dev), tf, proprio[t].to(dev))
    second = BatchedRollout(d, B, kv_bits=8)
    second.adopt(first)
    second.reset([1])
    for t, mode in ((3, "mixed"), (4, "cached"), (5, "cached")):
        got = second.step(images[t].reshape(B * 2, 3, 112, 112).to(dev), tf, proprio[t].to(dev)).cpu().double()
        assert second.last_mode == mode
        for e in range(B):
            assert float((got[e].reshape(-1) - _newest_action(second, sd, e, mc.transformer_heads)).abs().max()) <= 1e-4


def test_public_objects_take_the_setting(dev):
    """OTTER.kv_cache_bits and BatchedRolloutPolicy(kv_bits=...) run the same engine; the default keeps the fp32 history."""
    from otter_amd.engine import BatchedRollout
    from otter_amd.kv_cache import KVCache
    from otter_amd.rollout_server import BatchedRolloutPolicy
    model, sd, mc = _model(dev, 4, 53)
    images, proprio, text = _observations(6, 1, 31)
    model.kv_cache_bits = 8
    alone = BatchedRollout(model.device_model(), 1, kv_bits=8)
    tf = model.device_model().clip.text_tokens_cached(text)
    for t in range(6):
        a = model.forward_inference(images[t, 0].to(dev), text[0], proprio[t, 0].to(dev))
        b = alone.step(images[t, 0].to(dev), tf, proprio[t].to(dev))
        assert torch.equal(a, b[0])
    assert all(isinstance(c, KVCache) and c.bits == 8 for c in model._rollout._cache)
    pol = BatchedRolloutPolicy(model, 2, 2, kv_bits=4)
    frames = images[:2, 0].reshape(4, 3, 112, 112).to(dev)
    out = pol(frames, text.expand(2, -1).contiguous(), np.zeros((2, 6)), np.zeros(2))
    assert tuple(out.shape) == (2, 7) and bool(torch.isfinite(out).all()) and pol.rollout._cache[0].bits == 4
    model.invalidate_device_weights()
    pol.refresh()
    assert pol.rollout.kv_bits == 4 and pol.rollout._cache[0].bits == 4
    assert isinstance(BatchedRollout(model.device_model(), 1)._cache[0], torch.Tensor)


def test_captured_policy_steps_beside_eager_ones(dev):
    """A cached step of the policy captured into a graph before any eager one, replayed between eager steps of other batch sizes and positions:
    every replay gives what the eager step gives on the same history."""
    model, sd, mc = _model(dev, 8, 59)
    pol = model.device_model().policy
    g = torch.Generator().manual_seed(61)
    windows = {b: torch.randn(b, 8, pol.dim, generator=g).to(dev) for b in (2, 3)}
    cache, twin, other = (pol.new_cache(b, 8, 4) for b in (2, 2, 3))
    plain = pol.new_cache(2, 8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        pol.run(windows[2], plain, 1, 0)                        # (loads the kernels; no quantised cache yet)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = pol.run(windows[2], cache, 1, 1)
    for turn in range(4):
        windows[2].copy_(torch.randn(2, 8, pol.dim, generator=g))
        for c, t in zip(cache, twin):
            c.codes.zero_(), c.scales.zero_(), t.codes.zero_(), t.scales.zero_()
        pol.run(windows[2], cache, 1, 0)
        pol.run(windows[2], twin, 1, 0)
        pol.run(windows[3], other, 1, turn + 2)
        graph.replay()
        want = pol.run(windows[2], twin, 1, 1)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert all(torch.equal(c.codes, t.codes) and torch.equal(c.scales, t.scales) for c, t in zip(cache, twin))
