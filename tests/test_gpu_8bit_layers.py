"""Layers over pages of 8 bits on the GPU: a window, sinks, no norm, no rotation, a call that reads another call's pages, each
against the same layer on the host with plain kernels (tests/test_8bit_engine_cpu.py).

Float32: the two differ by float32 roundings, and where such a difference lies on a border between two steps of a page's values, by
that step (1/127 of the block's largest value) in one of thousands of values: most rows agree to 1e-4 of the largest, all to
2e-2.  bfloat16: the bound of the other layers' tests, 3e-2, and one step of 1/127 more."""
import random

import pytest
import torch

import toy
from rvllm_b200.cache import CacheManager
from rvllm_b200.engine import BatchBuilder, StepEntry, load_model
from rvllm_b200.parts import AttentionSpec, NormSpec, PositionSpec, mixer_class
from test_8bit_engine_cpu import Plain8
from test_8bit_layers_cpu import folder, replayed  # noqa: F401
from test_gpu_parts import tensors_for

pytestmark = pytest.mark.gpu


def near(got, want, dtype):
    scale = float(want.abs().max())
    error = (got - want).abs().amax(1) / scale
    if dtype in (torch.float32, "float32"):
        assert float(error.median()) <= 1e-4 and float(error.max()) <= 2e-2, (float(error.median()), float(error.max()))
    else:
        assert float(error.max()) <= 3e-2 + 1 / 127, float(error.max())


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("schedule", ["whole", "tail_decode", "portions", "mixed"])
def test_a_window_and_shared_pages(folder, dtype, schedule):  # noqa: F811
    want = replayed(load_model(folder, "float32", "cpu", Plain8())[0], schedule)
    got = replayed(load_model(folder, dtype, "cuda")[0], schedule)
    assert got.keys() == want.keys()
    near(torch.stack([got[k].float().cpu() for k in want]), torch.stack([want[k] for k in want]), dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,dim,window,norm,turn", [
    (6, 2, 48, 11, True, True), (8, 2, 64, 40, True, False), (4, 4, 64, None, False, True), (8, 1, 128, 70, False, False)])
def test_sinks_and_windows(dtype, heads, kv, dim, window, norm, turn):
    from rvllm_b200.kernels import cuda_ops
    hidden = 96
    spec = AttentionSpec("attention", hidden, num_heads=heads, num_kv_heads=kv, head_dim=dim, window=window, sinks=True,
                         qk_norm=NormSpec("rmsnorm", dim, 1e-5) if norm else None,
                         position=PositionSpec("rope", dim, 10000.0, 512) if turn else PositionSpec("none"))
    cls = mixer_class("attention")
    assert cls.eight_bit_cache(spec)
    dev, host = tensors_for(cls.params(spec), dtype)
    sides = [(cls(spec, dev, cuda_ops(), dtype), "cuda", dtype), (cls(spec, host, Plain8(), torch.float32), "cpu", torch.float32)]
    lengths, rng = [150, 9, 1, 83], random.Random(5)
    g = torch.Generator().manual_seed(3)
    xs = [(torch.randn(n, hidden, generator=g) * 2).bfloat16().float() for n in lengths]
    caches = [CacheManager([cls.cache_need(spec)], [None], 8, 64, len(lengths), dtype=d, device=where, kv_dtype=torch.int8)
              for _, where, d in sides]
    builders = [BatchBuilder(c, part.ops, where, pinned=where == "cuda") for c, (part, where, _) in zip(caches, sides)]
    for c in caches:
        for i in range(len(lengths)):
            c.add(i)
    done, rows = [0] * len(lengths), [[], []]
    while any(d < n for d, n in zip(done, lengths)):
        live = [(i, min(rng.choice([1, 1, 2, 5, 17, 60]), n - done[i])) for i, n in enumerate(lengths) if done[i] < n]
        live.sort(key=lambda e: e[1] != 1)
        for side, (cache, builder, (part, where, d)) in enumerate(zip(caches, builders, sides)):
            for i, take in live:
                cache.reserve(i, done[i] + take)
            ctx = builder.build([StepEntry(i, [0] * take, ()) for i, take in live])
            x = torch.cat([xs[i][done[i]:done[i] + take] for i, take in live]).to(where, d)
            rows[side].append(part.forward(x, ctx, cache.views()[0]).float().cpu())
            for i, take in live:
                cache.advance(i, done[i] + take)
        for i, take in live:
            done[i] += take
    near(torch.cat(rows[0]), torch.cat(rows[1]), dtype)
