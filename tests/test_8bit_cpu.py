"""What the calls of the 8-bit cache and of the log probabilities refuse, and that nothing is launched then, without a GPU:
the kernels are stand-ins that note their calls."""
from types import SimpleNamespace

import pytest
import torch

from rvllm_b200.errors import KernelError
from rvllm_b200.kernels import bindings
from rvllm_b200.kernels.bindings import CudaOps

F32, BF16, I8, I32 = torch.float32, torch.bfloat16, torch.int8, torch.int32


class OnDevice(torch.Tensor):
    """A tensor in host memory that says it is on a device."""

    def get_device(self):
        return getattr(self, "number", 0)


def there(*shape, dtype=F32, number=0):
    t = torch.zeros(shape, dtype=dtype).as_subclass(OnDevice)
    t.number = number
    return t


@pytest.fixture
def ops(monkeypatch):
    o = object.__new__(CudaOps)
    o.calls, o.launches, o._sm_count = [], 0, 148
    o._here = lambda: 0
    o._raw_stream = lambda device: 0
    o.decode_8bit = "auto"
    o.prefill_8bit, o.prefill_attention, o.widen_8bit_bytes, o._attn_libs = "auto", "auto", 1 << 30, {}
    o.lib = SimpleNamespace(rv_last_error=lambda: b"refused by the library")
    note = lambda *a: o.calls.append(a) or 0  # noqa: E731
    o._write_8bit = o._read_8bit = o._token_logprobs = o._widen_8bit = note
    o._attn8_lib = lambda d: (note, lambda *a: 0, lambda: b"refused by the library")
    o._attn5_wide = lambda d: (note, lambda: b"refused by the library")
    o._gemm_status = lambda d: there(1, dtype=I32)
    return o


def write_args(**change):
    a = dict(qkv=there(5, 8 * 64, dtype=BF16), num_heads=4, num_kv_heads=2, head_dim=64, q_weight=there(64), k_weight=there(64),
             eps=1e-6, table=(there(99, 32), there(99, 32)), positions=there(5, dtype=I32), slot_mapping=there(5, dtype=I32),
             q_out=there(5, 256, dtype=BF16), k_cache=there(7, 2, 16, 64, dtype=I8), v_cache=there(7, 2, 16, 64, dtype=I8),
             k_scale=there(7, 2), v_scale=there(7, 2))
    return {**a, **change}


@pytest.mark.parametrize("change", [
    {}, dict(table=None, positions=None), dict(q_weight=None, k_weight=None), dict(qkv=there(5, 600, dtype=BF16)),
    dict(qkv=there(0, 512, dtype=BF16), q_out=there(0, 256, dtype=BF16)), dict(slot_mapping=there(9, dtype=I32))])
def test_write_takes(ops, change):
    ops.qk_norm_rope_write_8bit(**write_args(**change))
    assert len(ops.calls) == 1 and ops.launches == 1


@pytest.mark.parametrize("change", [
    dict(qkv=there(5, 512, dtype=torch.float16)), dict(qkv=there(5, 511, dtype=BF16)), dict(qkv=there(5, 1024, dtype=BF16)[:, ::2]),
    dict(qkv=there(1, 512, dtype=BF16).expand(5, 512)), dict(qkv=there(5, 512, dtype=BF16, number=1)), dict(qkv=there(5, 512)),
    dict(num_heads=0), dict(num_kv_heads=0), dict(num_kv_heads=1), dict(head_dim=32),
    dict(q_weight=there(32)), dict(k_weight=there(64, dtype=BF16)), dict(k_weight=there(64, number=1)),
    dict(table=(there(99, 64), there(99, 64))), dict(table=(there(99, 32), there(98, 32))), dict(table=(there(99, 32), there(99, 32, number=1))),
    dict(positions=there(4, dtype=I32)), dict(positions=there(5, dtype=torch.int64)), dict(slot_mapping=there(4, dtype=I32)),
    dict(slot_mapping=there(5, dtype=torch.int64)), dict(slot_mapping=there(10, dtype=I32)[::2]),
    dict(q_out=there(5, 512, dtype=BF16)), dict(q_out=there(4, 256, dtype=BF16)), dict(q_out=there(5, 256)),
    dict(q_out=there(5, 512, dtype=BF16)[:, :256]), dict(q_out=there(5, 256, dtype=BF16, number=1)),
    dict(k_cache=there(7, 2, 16, 64, dtype=torch.uint8)), dict(k_cache=there(7, 16, 2, 64, dtype=I8).transpose(1, 2)),
    dict(k_cache=there(6, 2, 16, 64, dtype=I8)), dict(v_cache=there(7, 2, 8, 64, dtype=I8)), dict(v_cache=there(7, 2, 16, 64, dtype=I8, number=1)),
    dict(k_scale=there(7, 1)), dict(k_scale=there(7, 2, dtype=BF16)), dict(v_scale=there(2, 7).t()),
    dict(k_cache=there(7, 2, 1024, dtype=I8)),
    dict(qkv=there(5, 8 * 40, dtype=BF16), head_dim=40, q_out=there(5, 160, dtype=BF16), table=None, q_weight=None, k_weight=None,
         k_cache=there(7, 2, 16, 40, dtype=I8), v_cache=there(7, 2, 16, 40, dtype=I8)),
    dict(qkv=there(5, 8 * 272, dtype=BF16), head_dim=272, q_out=there(5, 1088, dtype=BF16), table=None, q_weight=None, k_weight=None,
         k_cache=there(7, 2, 16, 272, dtype=I8), v_cache=there(7, 2, 16, 272, dtype=I8))])
def test_write_refuses(ops, change):
    with pytest.raises(KernelError, match="write_8bit|float32 or bfloat16"):
        ops.qk_norm_rope_write_8bit(**write_args(**change))
    assert not ops.calls


@pytest.mark.parametrize("cache,scale,pages,dtype", [
    (there(7, 2, 16, 64), there(7, 2), there(3, dtype=I32), BF16), (there(7, 2, 16, 64, dtype=I8), there(7, 3), there(3, dtype=I32), BF16),
    (there(7, 2, 16, 64, dtype=I8), there(7, 2), there(3, dtype=torch.int64), BF16),
    (there(7, 2, 16, 64, dtype=I8), there(7, 2), there(3, 1, dtype=I32), BF16),
    (there(7, 2, 16, 64, dtype=I8), there(7, 2), there(3, dtype=I32), torch.float16),
    (there(7, 2, 16, 8, dtype=I8), there(7, 2), there(3, dtype=I32), F32),
    (there(7, 2, 16, 64, dtype=I8, number=1), there(7, 2), there(3, dtype=I32), F32)])
def test_read_refuses(ops, cache, scale, pages, dtype):
    with pytest.raises(KernelError):
        ops.read_8bit(cache, scale, pages, dtype)
    assert not ops.calls


def attend_args(change=None, ctx=None, group=None):
    c = dict(n_reqs=3, n_tokens=6, n_decode=2, q_start=there(4, dtype=I32), ctx_lens=there(3, dtype=I32), max_q_len=4, max_ctx_len=99)
    g = dict(block_table=there(3, 8, dtype=I32), page_size=16)
    a = dict(q=there(6, 256, dtype=BF16), num_heads=4, num_kv_heads=2, head_dim=64, k_cache=there(7, 2, 16, 64, dtype=I8),
             v_cache=there(7, 2, 16, 64, dtype=I8), k_scale=there(7, 2), v_scale=there(7, 2),
             ctx=SimpleNamespace(**{**c, **(ctx or {})}), group=SimpleNamespace(**{**g, **(group or {})}), scale=0.125, window=None,
             out=there(6, 256, dtype=BF16), sinks=None)
    return {**a, **(change or {})}


def test_attention_takes(ops):
    for change in ({}, dict(window=0), dict(window=7, sinks=there(4)), dict(q=there(6, 300, dtype=BF16)),
                   dict(q=there(6, 256), out=there(6, 256)), dict(q=there(9, 256, dtype=BF16), out=there(9, 256, dtype=BF16))):
        ops.calls.clear()
        ops.paged_attention_8bit(**attend_args(change))
        assert len(ops.calls) == 1


@pytest.mark.parametrize("change,ctx,group", [
    (dict(num_heads=3), {}, {}), (dict(num_heads=0), {}, {}), (dict(num_kv_heads=1), {}, {}), (dict(head_dim=32), {}, {}),
    (dict(q=there(6, 255, dtype=BF16)), {}, {}), (dict(q=there(6, 256, dtype=torch.float16)), {}, {}), (dict(q=there(6, 256)), {}, {}),
    (dict(q=there(5, 256, dtype=BF16)), {}, {}), (dict(q=there(6, 512, dtype=BF16)[:, ::2]), {}, {}),
    (dict(q=there(6, 256, dtype=BF16, number=1)), {}, {}),
    (dict(out=there(6, 255, dtype=BF16)), {}, {}), (dict(out=there(6, 512, dtype=BF16)[:, :256]), {}, {}),
    (dict(k_cache=there(7, 2, 16, 64, dtype=BF16)), {}, {}), (dict(v_cache=there(8, 2, 16, 64, dtype=I8)), {}, {}),
    (dict(k_scale=there(2, 7)), {}, {}), (dict(v_scale=there(7, 2, number=1)), {}, {}),
    (dict(window=-1), {}, {}), (dict(sinks=there(3)), {}, {}), (dict(sinks=there(4, dtype=BF16)), {}, {}),
    ({}, dict(n_decode=4), {}), ({}, dict(n_decode=-1), {}), ({}, dict(n_tokens=1), {}), ({}, dict(n_tokens=7), {}),
    ({}, dict(q_start=there(3, dtype=I32)), {}), ({}, dict(ctx_lens=there(2, dtype=I32)), {}),
    ({}, dict(ctx_lens=there(3, dtype=torch.int64)), {}), ({}, {}, dict(page_size=8)),
    ({}, {}, dict(block_table=there(2, 8, dtype=I32))), ({}, {}, dict(block_table=there(3, 16, dtype=I32)[:, ::2])),
    ({}, {}, dict(block_table=there(24, dtype=I32))), ({}, {}, dict(block_table=there(3, 8, dtype=I32, number=1)))])
def test_attention_refuses(ops, change, ctx, group):
    with pytest.raises(KernelError, match="attention_8bit|float32 or bfloat16"):
        ops.paged_attention_8bit(**attend_args(change, ctx, group))
    assert not ops.calls


def test_which_kernel_takes_portions(ops):
    """Long bfloat16 portions with heads of 64 or 128 are widened (two launches more than the single tokens'), others and such
    as would take more memory than they may are not; `prefill_8bit` forces either where it can."""
    def calls(tokens=2050, dtype=BF16, dim=64, stride=0, longest=2048, deepest=2048, n_decode=2, window=None):
        ops.calls.clear()
        wide = there(tokens, 4 * dim + stride, dtype=dtype)
        args = attend_args(dict(q=wide[:, :4 * dim], out=there(tokens, 4 * dim, dtype=dtype), head_dim=dim, window=window,
                                k_cache=there(7, 2, 16, dim, dtype=I8), v_cache=there(7, 2, 16, dim, dtype=I8)),
                           dict(n_tokens=tokens, max_q_len=longest, max_ctx_len=deepest, n_decode=n_decode))
        args["q"].number = 0
        ops.paged_attention_8bit(**args)
        return len(ops.calls)
    assert calls() == 3 and calls(dim=128) == 3 and calls(n_decode=0) == 2 and calls(stride=64) == 3
    assert calls(dtype=F32) == 1 and calls(dim=80) == 1 and calls(stride=8) == 1 and calls(tokens=6, longest=4, deepest=99) == 1
    assert calls(deepest=1 << 23) == 1 and calls(deepest=1 << 23, window=1000) == 3
    ops.prefill_8bit = "rows"
    assert calls() == 1
    ops.prefill_8bit = "tcgen05"
    assert calls(tokens=6, longest=4, deepest=99) == 3 and calls(dtype=F32) == 1


@pytest.mark.parametrize("logits,tokens,top", [
    (there(3, 9, dtype=torch.float16), there(3, dtype=I32), 0), (there(3, 9), there(3, dtype=torch.int64), 0),
    (there(3, 9), there(2, dtype=I32), 0), (there(3, 9), there(3, 1, dtype=I32), 0), (there(3, 9), there(3, dtype=I32), 10),
    (there(3, 99), there(3, dtype=I32), 33), (there(3, 9), there(3, dtype=I32), -1), (there(3, 0), there(3, dtype=I32), 0),
    (there(27), there(3, dtype=I32), 0), (there(9, 3).t(), there(3, dtype=I32), 0), (there(1, 9).expand(3, 9), there(3, dtype=I32), 0),
    (there(3, 9, number=1), there(3, dtype=I32), 0), (there(3, 9), there(3, dtype=I32, number=1), 0)])
def test_logprobs_refuse(ops, logits, tokens, top):
    with pytest.raises(KernelError, match="token_logprobs|float32 or bfloat16"):
        ops.token_logprobs(logits, tokens, top)
    assert not ops.calls


def test_a_code_from_the_library_is_an_error(ops):
    ops._write_8bit = ops._token_logprobs = lambda *a: 1
    ops._attn8_lib = lambda d: (lambda *a: 1, lambda *a: 0, lambda: b"refused by the library")
    for call in (lambda: ops.qk_norm_rope_write_8bit(**write_args()), lambda: ops.paged_attention_8bit(**attend_args()),
                 lambda: ops.token_logprobs(there(3, 9), there(3, dtype=I32), 2)):
        with pytest.raises(KernelError, match="refused by the library"):
            call()


def test_records_hold_what_the_library_reads():
    """8 bytes an argument: addresses, whole numbers, a real number last."""
    assert [r.size for r in (bindings._WRITE_8BIT, bindings._READ_8BIT, bindings._ATTEND_8BIT, bindings._LOGPROBS)] == [184, 88, 232, 104]
