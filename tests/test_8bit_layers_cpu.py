"""Which layers hold keys and values in 8 bits, and what they compute from them, on the host: the plain kernels of
tests/test_8bit_engine_cpu.py under the toy architecture of tests/toy.py (a window, no norm and no rotation, a call that reads another
call's pages, blocks that keep a state and no pages)."""
import dataclasses
import os
import random

import pytest
import torch

import schedules
import toy
from plain_lfm2 import read_safetensors
from rvllm_b200.config import config_from_dict
from rvllm_b200.engine import ModelRunner, load_model, make_cache
from rvllm_b200.parts.model import Model
from rvllm_b200.weights import write_random_model
from test_8bit_engine_cpu import Plain8


@pytest.fixture(scope="module")
def folder(tmp_path_factory):
    toy.register_toy()
    return write_random_model(str(tmp_path_factory.mktemp("toy")), config_from_dict(toy.TOY), 7)


@pytest.fixture
def model(folder):
    return load_model(folder, "float32", "cpu", Plain8())[0]


def with_shift(model, layer):
    """The model's spec with a token shift before one block's mixer."""
    layers = list(model.spec.layers)
    layers[layer] = dataclasses.replace(layers[layer], token_shift=f"blocks.{layer}.shift")
    return dataclasses.replace(model.spec, layers=tuple(layers))


class Needs:
    """What `make_cache` asks of a model."""

    def __init__(self, model, spec):
        self.spec, self.dtype, self.device = spec, model.dtype, model.device
        self.cache_needs = lambda: Model.cache_needs(self)


def test_a_layer_without_pages_is_no_hindrance(model):
    """A mixer that keeps a state is not asked for keys and values in 8 bits, within a token shift (whose block keeps a second state)
    no more than by itself; one with pages within a token shift holds them so."""
    for layer in (0, 3):
        cache = make_cache(Needs(model, with_shift(model, layer)), 4, 16, 2, "int8")
        assert cache.eight_bit and all(g.k.dtype == torch.int8 for g in cache.groups) and len(cache.states) > 2
    cache = make_cache(Needs(model, with_shift(model, 3)), 4, 16, 2, "int8")
    assert len(cache.groups) == 2


def replayed(model, schedule):
    """Logits of five requests under a schedule of tests/schedules.py, by request and position."""
    rng = random.Random(2)
    reqs = {f"t{i}": [rng.randrange(300) for _ in range(n)] for i, n in enumerate((40, 3, 77, 21, 50))}
    steps = schedules.tail_decode(reqs, 12) if schedule == "tail_decode" else getattr(schedules, schedule)(reqs)
    cache = make_cache(model, 8, schedules.tokens_held(steps, 64) // 8, 4, "int8")
    got = schedules.replay(ModelRunner(model, cache, model.ops), steps)
    assert all(g.pool.in_use == 0 for g in cache.groups)
    return got


@pytest.mark.parametrize("schedule", ["whole", "tail_decode", "portions", "mixed"])
def test_a_window_and_shared_pages_in_8_bits(folder, model, schedule):
    """Windowed pages given back, a call that owns no pages, no norm and no rotation: near the exact logits, whatever the cut (a
    value is off by half a step of its block's scale, 1/254 of the block's largest at least and 1/127 at most, and each growth of
    the scale adds as much: some hundredths of the largest logit)."""
    got = replayed(model, schedule)
    w = read_safetensors(os.path.join(folder, "model.safetensors"))
    rng = random.Random(2)
    for i, n in enumerate((40, 3, 77, 21, 50)):
        ids = [rng.randrange(300) for _ in range(n)]
        ref = toy.toy_plain_logits(ids, w, toy.TOY)
        for p in range(n):
            assert float((got[(f"t{i}", p)] - ref[p]).abs().max()) <= 0.1 * float(ref.abs().max()), (i, p)
