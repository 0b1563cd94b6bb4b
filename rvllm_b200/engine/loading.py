"""From a model folder to a runnable model: config.json picks the architecture, the
architecture builds the `ModelSpec`, the loader reads the declared tensors, and the
generic `Model` is put together from the registered parts.  (The reference:
`Model::load`, src/weights.rs:300-448, then `Runtime::new`, src/runtime.rs:24-77.)
"""
from __future__ import annotations

import torch

from ..cache import CacheManager
from ..config.registry import architecture, load_config
from ..parts.base import PagedNeed, SeveralNeeds, arrangement_class, mixer_class
from ..parts.model import Model
from ..weights.loader import load_tensors, tensor_shapes

DTYPES = {"bfloat16": torch.bfloat16, "bf16": torch.bfloat16,
          "float32": torch.float32, "fp32": torch.float32}


def parse_dtype(name) -> torch.dtype:
    if isinstance(name, torch.dtype):
        if name not in (torch.bfloat16, torch.float32):
            raise ValueError(f"compute dtype must be bfloat16 or float32, got {name}")
        return name
    if name not in DTYPES:
        raise ValueError(f"unknown dtype {name!r} (known: bfloat16, float32)")
    return DTYPES[name]


def load_model(folder: str, dtype="bfloat16", device="cuda", ops=None):
    """(model, config) for the folder.  `ops` defaults to the CUDA kernel set, whose
    import fails loudly when the native library cannot be built or loaded."""
    dtype = parse_dtype(dtype)
    config = load_config(folder)
    complete = getattr(config, "with_tensor_shapes", None)
    if complete is not None:
        # sizes that no key names are taken from the tensor file's header
        config = complete(tensor_shapes(folder))
    spec = architecture(config.architecture).build_spec(config)
    if ops is None:
        from ..kernels import cuda_ops
        ops = cuda_ops()
    tensors = load_tensors(folder, spec, dtype, device)
    model = Model(spec, tensors, ops, dtype)
    del tensors
    return model, config


KV_CACHES = {"auto": None, "int8": torch.int8}


def parse_kv_cache(name):
    """None (keys and values in the model's type) or torch.int8."""
    if name is None or name == torch.int8:
        return name
    if name not in KV_CACHES:
        raise ValueError(f"unknown key/value cache {name!r} (known: auto, int8)")
    return KV_CACHES[name]


def _holds_pages(need) -> bool:
    if isinstance(need, SeveralNeeds):
        return any(_holds_pages(part) for part in need.parts)
    return isinstance(need, PagedNeed)


def make_cache(model: Model, page_size: int, num_pages: int, max_requests: int,
               kv_cache="auto") -> CacheManager:
    """`kv_cache` "int8": keys and values in 8 bits with a scale per page and head, for models whose
    attention layers all read such pages."""
    kv_dtype, needs = parse_kv_cache(kv_cache), model.cache_needs()
    if kv_dtype is not None:
        for call in model.spec.order:
            block = model.spec.layers[call.layer]
            need = arrangement_class(block.arrangement).cache_need(block)
            if _holds_pages(need) and not mixer_class(block.mixer.kind).eight_bit_cache(block.mixer):
                raise ValueError(f"a layer of kind {block.mixer.kind!r} as this model has it does not read "
                                 f"keys and values in 8 bits")
    return CacheManager(needs, [c.cache_of for c in model.spec.order],
                        page_size, num_pages, max_requests, dtype=model.dtype,
                        device=model.device, kv_dtype=kv_dtype)
