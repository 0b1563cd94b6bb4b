"""Which layers hold keys and values in 8 bits, and what they compute from them, on the host: the plain kernels of
tests/test_8bit_engine_cpu.py under the toy architecture of tests/toy.py (a window, no norm and no rotation, a call that reads another
call's pages, blocks that keep a state and no pages)."""
import dataclasses
import random

import pytest
import torch

import schedules
import toy
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
