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


class Pool:
    """A cache manager's live requests, as far as padding asks."""

    def __init__(self, page_size, computed):
        self.page_size = page_size
        self.requests = {r: SimpleNamespace(computed=n) for r, n in enumerate(computed)}


def engine_step(ops, new, old, page_size=16, H=32, K=8, D=64, dtype=BF16):  # noqa: F811
    """The attention call of a step of portions `new` after `old` tokens, padded as `ModelRunner` pads it: whether it is widened."""
    from rvllm_b200.engine import ModelRunner, StepEntry
    runner = object.__new__(ModelRunner)
    runner.cache, runner._portion_limits, runner._shallow = Pool(page_size, old), None, 0
    entries = sorted((StepEntry(r, range(n), (n - 1,)) for r, n in enumerate(new)), key=lambda e: len(e.tokens) != 1)
    key = runner._mixture_sizes(entries)
    singles, reqs, tokens, width, longest, deepest = key
    ops.calls.clear()
    ops.paged_attention_8bit(**attend_args(
        dict(q=there(tokens, H * D, dtype=dtype), out=there(tokens, H * D, dtype=dtype), num_heads=H, num_kv_heads=K, head_dim=D,
             k_cache=there(7, K, page_size, D, dtype=I8), v_cache=there(7, K, page_size, D, dtype=I8), k_scale=there(7, K), v_scale=there(7, K)),
        dict(n_reqs=singles + reqs, n_tokens=tokens, n_decode=singles, q_start=there(singles + reqs + 1, dtype=I32),
             ctx_lens=there(singles + reqs, dtype=I32), max_q_len=longest, max_ctx_len=deepest, likely=runner._likely(key)),
        dict(block_table=there(singles + reqs, width, dtype=I32), page_size=page_size)))
    return any(len(c) > 20 for c in ops.calls)         # (the record of the other kernel is one argument)


@pytest.mark.parametrize("new,old,H,K,D,widened", [
    ([64], [0], 32, 8, 64, False), ([64], [1000], 32, 8, 64, True), ([64], [6000], 32, 8, 64, True), ([256], [0], 32, 8, 64, True),
    ([512], [0], 32, 8, 64, True), ([2048], [0], 32, 8, 64, True), ([256], [1000], 16, 2, 128, True), ([64], [500], 16, 8, 64, False),
    ([20] * 8, [500] * 8, 32, 8, 64, False), ([10] * 16, [1500] * 16, 32, 8, 64, False), ([40] * 16, [500] * 16, 32, 8, 64, True),
    ([10] * 32, [1500] * 32, 16, 8, 64, False), ([10] * 16, [500] * 16, 16, 2, 128, False), ([512] * 4, [1000] * 4, 32, 8, 64, True),
    ([100] + [1] * 8, [300] * 9, 32, 8, 64, False), ([100] + [1] * 8, [3000] * 9, 32, 8, 64, True),
    ([100] + [1] * 31, [1000] * 32, 16, 2, 128, False), ([500] + [1] * 31, [2000] * 32, 32, 8, 64, True)])
def test_padded_steps_choose_by_what_is_there(ops, new, old, H, K, D, widened):  # noqa: F811
    """An engine's step counts an empty portion more, all tokens as one portion and the next power of two of pages; the choice
    follows what a step of these sizes has, not what its launches have to cover, and is the kernel that such a step was measured to be
    faster with."""
    assert engine_step(ops, new, old, H=H, K=K, D=D) == widened


def test_sizes_alone_say_what_is_likely():
    from rvllm_b200.engine import ModelRunner
    runner = object.__new__(ModelRunner)
    runner.cache = Pool(16, [])
    assert runner._likely((0, 2, 64, 128, 64, 2048)) == (64, 1, 1536)
    assert runner._likely((32, 4, 2048, 16, 2016, 64)) == (2016, 2, 64)
    assert runner._likely((64, 2, 64, 16, 1, 256)) == (1, 1, 192)


def test_portions_are_widened_as_many_at_a_time_as_may_be(ops):  # noqa: F811
    """Many portions of long contexts need not all be widened at once: each pass has those that the limit holds, and names the requests,
    lengths and first tokens that are its own."""
    q_start, lens = there(8, dtype=I32), there(7, dtype=I32)
    q_start[:], lens[:] = torch.tensor([0, 1, 2, 514, 1026, 1538, 2050, 2050]), torch.tensor([9, 9, 4096, 4000, 3000, 2000, 0])
    args = lambda: attend_args(dict(q=there(2050, 256, dtype=BF16), out=there(2050, 256, dtype=BF16)),  # noqa: E731
                               dict(n_reqs=7, n_tokens=2050, max_q_len=512, max_ctx_len=4096, n_decode=2, q_start=q_start, ctx_lens=lens),
                               dict(block_table=there(7, 256, dtype=I32)))
    a_portion = 4 * 4096 * 2 * 64
    for limit, passes in ((5 * a_portion, [5]), (5 * a_portion - 1, [4, 1]), (2 * a_portion, [2, 2, 1]), (a_portion, [1] * 5), (a_portion - 1, None)):
        ops.calls.clear()
        ops.widen_8bit_bytes = limit
        ops.paged_attention_8bit(**args())
        if passes is None:
            assert len(ops.calls) == 1
            continue
        assert len(ops.calls) == 1 + 2 * len(passes)
        first = 2
        for widen, attend, n in zip(ops.calls[1::2], ops.calls[2::2], passes):
            assert widen[17:19] == (first, n) and attend[11:13] == (0, n)
            assert attend[8] == q_start.data_ptr() + 4 * first and attend[9] == lens.data_ptr() + 4 * first
            first += n


def test_without_memory_the_pages_are_read_as_they_are(ops, monkeypatch):  # noqa: F811
    """Copies that find no memory are no error: the kernel that needs none takes the portions."""
    assert portions(ops) == 3
    real = torch.empty

    def empty(*a, **k):
        if k.get("dtype") == BF16:
            raise torch.cuda.OutOfMemoryError("no memory left")
        return real(*a, **k)

    monkeypatch.setattr(torch, "empty", empty)
    args = attend_args(dict(q=there(2050, 256, dtype=BF16), out=there(2050, 256, dtype=BF16)),
                       dict(n_tokens=2050, max_q_len=2048, max_ctx_len=2048, n_decode=2))
    ops.calls.clear()
    ops.paged_attention_8bit(**args)
    assert len(ops.calls) == 1
