"""Generation, scoring and replayed steps with keys and values in 8 bits, and log probabilities, on the GPU.

The comparison is the same engine on the host with plain kernels (tests/test_8bit_engine_cpu.py).  Float32: the two differ by float32
roundings, and where such a difference lies on a border between two steps of a page's values, by that step (1/127 of the
block's largest value) in one of thousands of values: most logits agree to 1e-4 of the largest, all to 2e-2.
bfloat16: the bound of the other models' tests, 3e-2."""
import os

import pytest
import torch

from rvllm_b200 import GenerateOptions, Generator
from rvllm_b200.engine import ModelRunner, StepEntry, load_model, make_cache
from test_8bit_engine_cpu import Plain8
from tiny import write_tiny

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    root = str(tmp_path_factory.mktemp("models"))
    return {"A": write_tiny(root, "A"), "B": write_tiny(root, "B"),
            "wide": write_tiny(os.path.join(root, "wide"), "A", hidden_size=128, num_attention_heads=8, num_key_value_heads=2, head_dim=64)}


def steps_of(folder, device, dtype, ops=None, graphs=False, cuts=((23, 9), (1, 30), (1, 1), (1, 1), (5, 1), (1, 1), (1, 1))):
    """Logits of two requests that bring `cuts` tokens a step, single tokens beside portions."""
    model, _ = load_model(folder, dtype, device, ops=ops)
    runner = ModelRunner(model, make_cache(model, 8, 40, 2, "int8"), model.ops, use_graphs=graphs)
    out, at = [], [0, 0]
    for r in (0, 1):
        runner.add_request(r)
    for cut in cuts:
        entries = [StepEntry(r, [(37 * i + 11 + 91 * r) % 500 for i in range(at[r], at[r] + n)], range(n)) for r, n in enumerate(cut)]
        out.append(runner.step(entries).float().cpu())
        at = [a + n for a, n in zip(at, cut)]
    if hasattr(model.ops, "check_status"):
        model.ops.check_status()
    return torch.cat(out), runner


@pytest.mark.parametrize("name", ["A", "B", "wide"])
@pytest.mark.parametrize("graphs", [False, True])
def test_steps(folders, name, graphs):
    want, _ = steps_of(folders[name], "cpu", "float32", Plain8())
    scale = float(want.abs().max())
    got, runner = steps_of(folders[name], "cuda", "float32", graphs=graphs)
    error = (got - want).abs().amax(1) / scale
    assert float(error.median()) <= 1e-4 and float(error.max()) <= 2e-2, (float(error.median()), float(error.max()))
    if graphs:
        assert runner.graph_steps > 0 and runner.capture_failures == 0
    half, _ = steps_of(folders[name], "cuda", "bfloat16", graphs=graphs)
    assert float((half - want).abs().max()) <= 3e-2 * scale


def test_score(folders):
    ids = [(29 * i + 3) % 500 for i in range(200)]
    for kv_cache in ("auto", "int8"):
        gen = Generator.load(folders["wide"], dtype="float32", kv_cache=kv_cache)
        got = gen.score(ids, top=3, portion=64)
        model, config = load_model(folders["wide"], "float32", "cpu", ops=Plain8())
        want = Generator(model, config, None, kv_cache).score(ids, top=3, portion=64)
        assert [t.token for t in got] == ids[1:]
        errors = sorted(abs(a.logprob - b.logprob) for a, b in zip(got, want))
        assert errors[len(errors) // 2] <= 1e-4 and errors[-1] <= 5e-2
        assert sum(a.rank == b.rank for a, b in zip(got, want)) >= 0.9 * len(got)
        assert all(abs(a.entropy - b.entropy) <= 5e-2 for a, b in zip(got, want))
        # (a shape that came before is replayed with the sizes of its padded block table: other splits, other roundings)
        assert all(abs(a.logprob - b.logprob) <= 1e-5 for a, b in zip(gen.score(ids, top=3, portion=64), got))


@pytest.mark.parametrize("kv_cache,dtype", [("auto", "float32"), ("int8", "float32"), ("int8", "bfloat16")])
@pytest.mark.parametrize("lookahead", [False, True])
def test_generation_with_logprobs(folders, kv_cache, dtype, lookahead):
    """Requests of several lengths, replayed steps, with and without the next step launched ahead: each token's own
    log probability, the most probable one under greedy sampling, and what scoring the whole text gives (float32: to 1e-3; in 8
    bits the pages of a text written whole differ by what growing scales drop)."""
    gen = Generator.load(folders["wide"], dtype=dtype, kv_cache=kv_cache)
    gen.lookahead = lookahead
    prompts = [[(7 * i + j) % 500 for i in range(n)] for j, n in enumerate((5, 17, 31, 60))]
    result = gen.generate_ids(prompts, GenerateOptions(max_tokens=20, block_size=8, stop_tokens=[], logprobs=4))
    for i, p in enumerate(prompts):
        lps = result.logprobs[i]
        assert [t.token for t in lps] == result.outputs[i] and len(lps) == 20
        assert all(t.rank == 1 and t.top[0][0] == t.token and len(t.top) == 4 for t in lps)
        scored = gen.score(p + result.outputs[i], block_size=8)[len(p) - 1:]
        bound = 1e-3 if kv_cache == "auto" else 0.2
        assert all(abs(a.logprob - b.logprob) <= bound for a, b in zip(lps, scored))
    again = gen.generate_ids(prompts, GenerateOptions(max_tokens=20, block_size=8, stop_tokens=[]))
    assert again.outputs == result.outputs and again.logprobs is None


def test_preemption_in_8_bits(folders):
    """A pool too small for all requests: recomputed ones get the tokens they get alone, or (as recomputed pages hold what one
    pass leaves) tokens that are as probable but for the pages' steps."""
    gen = Generator.load(folders["A"], dtype="float32", kv_cache="int8")
    prompts = [[(13 * i + j) % 500 for i in range(n)] for j, n in enumerate((5, 17, 31))]
    opts = dict(max_tokens=16, block_size=8, stop_tokens=[], logprobs=0)
    free = gen.generate_ids(prompts, GenerateOptions(**opts))
    tight = gen.generate_ids(prompts, GenerateOptions(num_blocks=9, prefill_chunk=6, **opts))
    assert tight.stats.preemptions > 0
    for i in range(3):
        assert len(tight.outputs[i]) == 16 and len(free.outputs[i]) == 16
        assert all(t.logprob <= 0 and t.rank == 1 for t in tight.logprobs[i])
    gen._runner.cache.check()


def test_command_line(folders, capsys):
    from rvllm_b200.cli import main
    assert main(["cli", "--model", folders["wide"], "--kv-cache", "int8", "--token-ids", "--prompt", "5 17 3", "--max-tokens", "4"]) == 0
    assert len(capsys.readouterr().out.split()) <= 4
