"""How the calls over pages of 8 bits choose their kernels, without a GPU: the kernels are stand-ins that note their calls."""
from types import SimpleNamespace

import pytest
import torch

from rvllm_b200.errors import KernelError
from test_8bit_cpu import BF16, F32, I8, I32, attend_args, ops, there  # noqa: F401


def portions(ops, **change):  # noqa: F811
    """Kernels launched for a portion of 2,048 tokens beside two single tokens: 3 where it is widened, else 1."""
    ops.calls.clear()
    args = attend_args(dict(q=there(2050, 256, dtype=BF16), out=there(2050, 256, dtype=BF16)),
                       dict(n_tokens=2050, max_q_len=2048, max_ctx_len=2048, n_decode=2, **change))
    ops.paged_attention_8bit(**args)
    return len(ops.calls)


@pytest.mark.parametrize("switch", ["mma", "simt"])
def test_the_switch_of_prompt_attention_holds_here_too(ops, switch):  # noqa: F811
    """Who keeps prompts off the tcgen05 kernel keeps those over 8-bit pages off it, unless these have been sent there by name."""
    assert portions(ops) == 3
    ops.prefill_attention = switch
    assert portions(ops) == 1
    ops.prefill_8bit = "tcgen05"
    assert portions(ops) == 3
    ops.prefill_attention, ops.prefill_8bit = "tcgen05", "rows"
    assert portions(ops) == 1


@pytest.mark.parametrize("name", ["decode_8bit", "prefill_8bit"])
def test_unknown_forms_are_refused(ops, name):  # noqa: F811
    setattr(ops, name, "fast")
    with pytest.raises(KernelError, match="paged_attention_8bit: .*fast"):
        portions(ops)
    assert not ops.calls
