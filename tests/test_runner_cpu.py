"""What the step function does when a launch sequence cannot be captured, on the host: the graphs are stand-ins."""
import pytest
import torch

from plain_ops import PlainOps
from rvllm_b200 import GenerateOptions
from rvllm_b200.engine import ModelRunner, StepEntry, load_model, make_cache
from rvllm_b200.engine import runner as runner_module
from test_8bit_engine_cpu import generator
from tiny import write_tiny


@pytest.fixture(scope="module")
def folder(tmp_path_factory):
    return write_tiny(str(tmp_path_factory.mktemp("models")), "A")


@pytest.fixture
def model(folder):
    return load_model(folder, "float32", "cpu", PlainOps())[0]


def portions(runner, lengths, start=0):
    """Logits of the last token of a request of each length, one step."""
    ids = [f"{start}-{i}" for i in range(len(lengths))]
    for r in ids:
        runner.add_request(r)
    out = runner.step([StepEntry(r, [(7 * j + 3 * i) % 500 for j in range(n)], (n - 1,)) for i, (r, n) in enumerate(zip(ids, lengths))])
    for r in ids:
        runner.end_request(r)
    return out


@pytest.mark.parametrize("kind", ["_MixedGraph", "_ShapeGraph"])
def test_a_capture_that_fails_leaves_the_step_to_its_launches(model, monkeypatch, kind):
    """A capture that ends in an error (no memory, a call that cannot be captured) costs a warning; this step and later ones of its
    sizes run without it."""
    tried = []

    class Fails:
        graph, broken, capturing, last_used = None, False, False, 0

        def __init__(self, runner, *key):
            pass

        def run(self, entries, row_order=None):
            tried.append(len(entries))
            self.capturing = True
            raise torch.cuda.OutOfMemoryError("no memory left")

    monkeypatch.setattr(runner_module, kind, Fails)
    cache = lambda: make_cache(model, 8, 32, 3)  # noqa: E731
    runner, plain = ModelRunner(model, cache(), model.ops), ModelRunner(model, cache(), model.ops)
    runner.use_graphs = True
    if kind == "_ShapeGraph":
        runner.max_mixed_graphs = -1
    for k in range(4):
        lengths = (9, 14)
        if k == 1:                                     # the second step of these sizes
            with pytest.warns(UserWarning, match="capturing a graph"):
                got = portions(runner, lengths, k)
        else:
            got = portions(runner, lengths, k)
        assert torch.allclose(got, portions(plain, lengths, k), atol=1e-5)
    assert tried == [2] and runner.capture_failures == 1 and runner.graph_steps == 0
    runner.cache.check()


class Replays:
    """A capture that launches its step kernel by kernel."""

    def __init__(self, runner, key, block_bucket):
        self.runner, self.key, self.width = runner, key, block_bucket
        self.graph, self.broken, self.capturing, self.last_used = object(), False, False, 0

    def run(self, entries, row_order=None):
        ctx = self.runner.builder.build(entries, pad_blocks=self.width, row_order=row_order)
        return self.runner.model.forward(ctx, self.runner.cache.views())


def test_scoring_captures_whole_portions_alone(folder, monkeypatch):
    """A text's last portion has a length of its own: a capture of each would hold the logits of all its tokens, and a place that other
    steps' captures want."""
    gen = generator(folder)
    ids = [(29 * i + 3) % 500 for i in range(40)]
    first = gen.score(ids, portion=13)
    for kind in ("_DecodeGraph", "_MixedGraph"):
        monkeypatch.setattr(runner_module, kind, lambda *a: pytest.fail("a capture"))
    monkeypatch.setattr(runner_module, "_ShapeGraph", Replays)
    runner = gen._runner
    runner.use_graphs = True
    for n in (40, 40, 33, 33, 36, 36, 20, 20):
        got = gen.score(ids[:n], portion=13)
        assert all(abs(a.logprob - b.logprob) <= 1e-5 and a.rank == b.rank for a, b in zip(got, first)) and len(got) == n - 1
    assert [k[0] for k in runner._shape_graphs] == [(13,)] and runner.graph_steps > 0
    runner.use_graphs = False
    assert gen.generate_ids([ids], GenerateOptions(max_tokens=2, stop_tokens=[])).outputs[0]


def test_captures_of_exact_shapes_are_bounded(model, monkeypatch):
    """By their number and by the logits that they keep; room is made by those that have not been replayed for a long time."""
    monkeypatch.setattr(runner_module, "_ShapeGraph", Replays)
    runner = ModelRunner(model, make_cache(model, 8, 32, 3), model.ops)
    runner.use_graphs, runner.max_mixed_graphs = True, -1
    runner.max_shape_logits = 20 * 4 * model.spec.vocab_size          # of twenty tokens

    def step(n, wanted):
        runner.add_request("r")
        runner.step([StepEntry("r", range(n), range(wanted))])
        runner.end_request("r")

    def twice(n, wanted):
        step(n, wanted)
        step(n, wanted)
        return [(k[0][0], len(k[1][0])) for k in runner._shape_graphs]

    assert twice(9, 9) == [(9, 9)] and twice(11, 11) == [(9, 9), (11, 11)]
    assert twice(12, 1) == [(9, 9), (11, 11)]                          # twenty are held
    assert twice(30, 30) == [(9, 9), (11, 11)]
    runner.mixed_graph_idle_steps = 8
    for _ in range(8):
        step(11, 11)
    assert twice(12, 1) == [(11, 11), (12, 1)]                         # the other one made room
    assert twice(30, 30) == [(11, 11), (12, 1)]                        # more than all may hold
    runner.max_shape_graphs, runner.max_shape_logits = 2, 1 << 40
    assert twice(14, 2) == [(11, 11), (12, 1)]
    runner.steps += 100
    step(12, 1)
    assert twice(15, 2) == [(12, 1), (15, 2)]
    runner.cache.check()


def test_more_alternatives_than_the_vocabulary_are_refused_before_a_step(folder, tmp_path):
    """As scoring refuses them: not by the kernel, when the first step has run and requests hold pages."""
    gen = generator(write_tiny(str(tmp_path), "A", vocab_size=20, bos_token_id=1, eos_token_id=7))
    for logprobs in (21, 32):
        with pytest.raises(ValueError, match="20"):
            gen.generate_ids([[1, 2, 3]], GenerateOptions(max_tokens=2, logprobs=logprobs))
    assert not gen._runner.cache.requests and gen._runner.steps == 0
    result = gen.generate_ids([[1, 2, 3]], GenerateOptions(max_tokens=2, logprobs=20, stop_tokens=[]))
    assert all(len(t.top) == 20 for t in result.logprobs[0])
