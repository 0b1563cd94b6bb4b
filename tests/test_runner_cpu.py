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


def test_scoring_captures_nothing(folder, monkeypatch):
    """Scoring wants a row of logits for every token: a launch sequence that kept them would hold them for good, one for every
    length of a text's last portion."""
    gen = generator(folder)
    ids = [(29 * i + 3) % 500 for i in range(40)]
    first = gen.score(ids, portion=13)
    for kind in ("_DecodeGraph", "_MixedGraph", "_ShapeGraph"):
        monkeypatch.setattr(runner_module, kind, lambda *a: pytest.fail("a capture"))
    gen._runner.use_graphs = True
    for _ in range(3):
        assert gen.score(ids, portion=13) == first
    assert not gen._runner._seen_shapes and not gen._runner._shape_graphs
    gen._runner.use_graphs = False
    assert gen.generate_ids([ids], GenerateOptions(max_tokens=2, stop_tokens=[])).outputs[0]

