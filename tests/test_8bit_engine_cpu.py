"""The engine with keys and values in 8 bits and with log probabilities, on the host: the plain kernels of tests/plain_ops.py
with the 8-bit calls and the log probabilities in 64 bits (tests/plain_8bit.py) beside them."""
import math

import pytest
import torch

import plain_8bit as plain
from plain_lfm2 import PlainModel
from plain_ops import PlainOps
from rvllm_b200 import GenerateOptions, Generator
from rvllm_b200.cache import CacheManager
from rvllm_b200.engine import ModelRunner, StepEntry, load_model, make_cache
from rvllm_b200.errors import CacheError
from rvllm_b200.parts.base import PagedNeed
from tiny import write_tiny


class Plain8(PlainOps):
    def qk_norm_rope_write_8bit(self, rows, H, K, D, qw, kw, eps, table, positions, slots, q_out, k8, v8, ks, vs):
        q, _, _ = plain.write(rows, H, K, D, qw, kw, eps, table, positions, slots, k8, v8, ks, vs)
        q_out.copy_(q)

    def paged_attention_8bit(self, q, H, K, D, k8, v8, ks, vs, ctx, group, scale, window, out, sinks=None):
        out.copy_(plain.attention(q, H, K, D, k8, v8, ks, vs, ctx, group, scale, window, sinks)[0])

    def token_logprobs(self, logits, tokens, top=0):
        rows = plain.logprobs(logits, tokens, top)
        f = lambda i: torch.tensor([r[i] for r in rows])  # noqa: E731
        return f(0).float(), f(1).int(), f(2).float(), f(3).float().reshape(len(rows), top), f(4).int().reshape(len(rows), top)


def generator(folder, kv_cache="auto", lookahead=False):
    model, config = load_model(folder, "float32", "cpu", ops=Plain8())
    gen = Generator(model, config, None, kv_cache)
    gen.lookahead = lookahead
    return gen


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    root = str(tmp_path_factory.mktemp("models"))
    return {n: write_tiny(root, n) for n in ("A", "B")}


def test_cache_manager_in_8_bits():
    m = CacheManager([PagedNeed(2, 64), PagedNeed(2, 64), PagedNeed(1, 32, window=9)], [None] * 3, 16, 5, 2, kv_dtype=torch.int8)
    first, second, third = m.views()
    assert first.k.dtype == first.v.dtype == torch.int8 and first.k.shape == (5, 2, 16, 64) and third.v.shape == (5, 1, 16, 32)
    assert first.k_scale.dtype == torch.float32 and first.k_scale.shape == (5, 2)
    assert first.k.is_contiguous() and second.v_scale.is_contiguous()
    first.k_scale[0, 0] = 1.0
    assert not second.k_scale.any() and not first.v_scale.any()
    # two heads of 64 in two layers, one of 32; scales: 8 bytes a page and head
    assert m.bytes_per_token() == 2 * 2 * (128 + 1) + (64 + 1)
    wide = CacheManager([PagedNeed(2, 64)], [None], 16, 5, 2)
    assert wide.views()[0].k_scale is None and wide.views()[0].k.shape == (5, 16, 2, 64)
    for need in (PagedNeed(1, 16, v_head_dim=32), PagedNeed(1, 16, values=False), PagedNeed(1, 16, every=4)):
        with pytest.raises(CacheError):
            CacheManager([need], [None], 16, 5, 2, kv_dtype=torch.int8)
    with pytest.raises(CacheError):
        CacheManager([PagedNeed(2, 64)], [None], 16, 5, 2, kv_dtype=torch.float16)


def test_kv_cache_is_refused_by_name_and_by_model(folders, tmp_path):
    with pytest.raises(ValueError, match="int8"):
        Generator.load(folders["A"], kv_cache="int4")
    import bizenex_tiny
    import vifanex_tiny
    for tiny in (bizenex_tiny, vifanex_tiny):
        model, _ = load_model(tiny.write(str(tmp_path), "A"), "float32", "cpu", ops=Plain8())
        with pytest.raises(ValueError, match="8 bits"):
            make_cache(model, 4, 8, 1, "int8")
        make_cache(model, 4, 8, 1)


@pytest.mark.parametrize("name", ["A", "B"])
def test_portions_and_tokens_agree_in_8_bits(folders, name):
    """A prompt whole, in portions and token by token leaves logits that differ by what the pages' growing scales drop: a
    step of 1/127 of a block's largest value, small beside the logits."""
    gen = generator(folders[name], "int8")
    ids = [(37 * i + 11) % 500 for i in range(41)]
    rows = {}
    for cut in (41, 13, 1):
        runner = ModelRunner(gen.model, make_cache(gen.model, 8, 8, 1, "int8"), gen.ops)
        runner.add_request("r")
        rows[cut] = torch.cat([runner.step([StepEntry("r", ids[a:a + cut], range(len(ids[a:a + cut])))]) for a in range(0, 41, cut)])
        runner.cache.check()
    exact = PlainModel(folders[name]).logits(ids)
    scale = float(exact.abs().max())
    for cut in rows:
        assert float((rows[cut] - rows[41]).abs().max()) <= 0.05 * scale
        assert float((rows[cut] - exact).abs().max()) <= 0.1 * scale and not torch.equal(rows[cut], exact)


def test_score(folders):
    gen = generator(folders["A"])
    ids = [(29 * i + 3) % 512 for i in range(30)]
    logits = PlainModel(folders["A"]).logits(ids).double()
    lp = torch.log_softmax(logits, 1)
    for portion in (512, 7, 1):
        got = gen.score(ids, top=3, portion=portion)
        assert [t.token for t in got] == ids[1:]
        for i, t in enumerate(got):
            assert abs(t.logprob - float(lp[i, ids[i + 1]])) <= 1e-4
            assert t.rank == int((logits[i] > logits[i, ids[i + 1]]).sum()) + 1
            assert abs(t.entropy + float((lp[i].exp() * lp[i]).sum())) <= 1e-4
            assert [a for a, _ in t.top] == torch.topk(lp[i], 3).indices.tolist()
    assert gen.score([5]) == [] and gen.score([]) == []
    assert not gen._runner.cache.requests
    for bad in (dict(prompt=[512]), dict(prompt=[1] * 300), dict(prompt=[1, 2], top=33), dict(prompt=[1, 2], portion=0)):
        with pytest.raises(ValueError):
            gen.score(**bad)


@pytest.mark.parametrize("kv_cache", ["auto", "int8"])
def test_logprobs_of_generated_tokens(folders, kv_cache):
    """Every output token has one, its own; under greedy sampling the most probable; preemption and portions change
    nothing of that."""
    gen = generator(folders["A"], kv_cache)
    prompts = [[(7 * i + j) % 512 for i in range(n)] for j, n in enumerate((5, 17, 31))]
    for opts in (dict(), dict(prefill_chunk=4, max_batched_tokens=9), dict(num_blocks=9, prefill_chunk=6)):
        result = gen.generate_ids(prompts, GenerateOptions(max_tokens=8, block_size=8, stop_tokens=[], logprobs=2, **opts))
        for i in range(3):
            lps = result.logprobs[i]
            assert [t.token for t in lps] == result.outputs[i] and len(lps) == 8
            assert all(t.rank == 1 and t.top[0] == (t.token, pytest.approx(t.logprob)) and t.logprob < 0 < t.entropy for t in lps)
    sampled = gen.generate_ids(prompts, GenerateOptions(max_tokens=8, temperature=1.5, seed=3, stop_tokens=[], logprobs=0))
    for i in range(3):
        assert [t.token for t in sampled.logprobs[i]] == sampled.outputs[i] and all(t.top == [] for t in sampled.logprobs[i])
    assert gen.generate_ids(prompts, GenerateOptions(max_tokens=2, stop_tokens=[])).logprobs is None
    with pytest.raises(ValueError):
        gen.generate_ids(prompts, GenerateOptions(max_tokens=2, logprobs=33))
    assert all(math.isfinite(t.logprob) for t in sampled.logprobs[0])
