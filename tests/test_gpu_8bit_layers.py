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


# ---- pages that change hands --------------------------------------------------------------------------------

@pytest.fixture(scope="module")
def wide(tmp_path_factory):
    from tiny import write_tiny
    return write_tiny(str(tmp_path_factory.mktemp("models")), "A", hidden_size=128, num_attention_heads=8, num_key_value_heads=2, head_dim=64)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_pages_that_change_hands(wide, dtype):
    """What a request's pages hold does not depend on who held them before: values, scales and logits are, bit for bit, those of a
    cache that is new, after every page has held larger values and smaller ones."""
    from rvllm_b200.engine import ModelRunner, make_cache
    model, _ = load_model(wide, dtype, "cuda")
    ids = [(37 * i + 11) % 500 for i in range(75)]
    cuts = [6, 6, 11, 1, 1, 1, 20, 6, 1, 1, 21]

    def run(runner):
        runner.add_request("r")
        logits, at = [], 0
        for n in cuts:
            logits.append(runner.step([StepEntry("r", ids[at:at + n], range(n))]).clone())
            at += n
        held = []
        table = torch.tensor(list(runner.cache.requests["r"].tables[0]), dtype=torch.int32, device="cuda")
        for view in runner.cache.views():
            if view is not None and view.kind == "paged":
                for pages, scale in ((view.k, view.k_scale), (view.v, view.v_scale)):
                    held += [model.ops.read_8bit(pages, scale, table, torch.float32).transpose(1, 2).flatten(0, 1)[:at],
                             scale[table.long()]]
        runner.end_request("r")
        return logits + held

    want = run(ModelRunner(model, make_cache(model, 8, 10, 1, "int8"), model.ops))
    runner = ModelRunner(model, make_cache(model, 8, 10, 1, "int8"), model.ops)
    for factor in (2.0 ** 9, 2.0 ** -30):
        run(runner)
        for group in runner.cache.groups:
            group.k_scale *= factor
            group.v_scale *= factor
            group.k.fill_(127)
            group.v.fill_(-127)
        again = run(runner)
        assert len(again) == len(want) and all(torch.equal(a, b) for a, b in zip(again, want))


def test_recomputed_requests_report_what_scoring_gives(wide):
    """A pool too small for all requests: what a preempted request reports for its tokens is what the whole text is scored at, to
    twice what cuts of a text differ by in 8 bits (0.05 of the largest logit each, as on the host)."""
    from rvllm_b200 import GenerateOptions, Generator
    gen = Generator.load(wide, dtype="float32", kv_cache="int8")
    prompts = [[(13 * i + j) % 500 for i in range(n)] for j, n in enumerate((5, 17, 31))]
    result = gen.generate_ids(prompts, GenerateOptions(num_blocks=9, prefill_chunk=6, max_tokens=16, block_size=8, stop_tokens=[], logprobs=3))
    assert result.stats.preemptions > 0
    gen._runner.add_request("r")
    largest = float(gen._runner.step([StepEntry("r", prompts[2], range(31))]).abs().max())
    gen._runner.end_request("r")
    for i, p in enumerate(prompts):
        out, lps = result.outputs[i], result.logprobs[i]
        scored = gen.score(p + out, top=3, block_size=8)[len(p) - 1:]
        assert [t.token for t in lps] == out == [t.token for t in scored]
        off = [abs(a.logprob - b.logprob) for a, b in zip(lps, scored)]
        assert max(off) <= 0.1 * largest, (max(off), largest)
    gen._runner.cache.check()


def test_command_line_prints_what_the_generator_gives(wide, capsys):
    from rvllm_b200 import GenerateOptions, Generator
    from rvllm_b200.cli import main
    want = Generator.load(wide, dtype="float32", kv_cache="int8").generate_ids([[5, 17, 3]], GenerateOptions(max_tokens=6)).outputs[0]
    assert main(["cli", "--model", wide, "--dtype", "float32", "--kv-cache", "int8", "--token-ids", "--prompt", "5 17 3", "--max-tokens", "6"]) == 0
    got = [int(t) for t in capsys.readouterr().out.split()]
    stop = [7] if want and want[-1] == 7 else []                      # (a stop token is not printed)
    assert got + stop == want and want
