"""Attention over pages of 8 bits at the edges of what its rows hold: queries of any size, queries with one large value beside
small ones, weights that nearly cancel, values of neighbouring pages far apart.  Each against the same in 64 bits
(tests/plain_8bit.py).

Tolerances.  The result's own rounding, `half` of itself (bfloat16 2^-8, float32 2^-24).  Scores come from float32 sums and
operands of 22 bits and more, weights from exponentials of 2^-22, and both enter the products with 22 bits: 2^-20 of the largest
value seen for each unit of the largest sum |q| |k| scale, and 8 units of them (as in `plain_8bit.attention_room`).  A weight
below 2^-8 of the row's reference has no more than the smallest step of its second part, 2^-25, beside a largest of 2^6: 2^-31 of
the largest term for each of `keys`, some sqrt(keys) of them together.  Portions that are widened multiply weights of float16,
half a step of which is 2^-11 of itself: as much of the largest value seen more."""
import math

import pytest
import torch

import plain_8bit as plain
from test_gpu_8bit import DTYPES, check_attention, ops, pages_of, rnd  # noqa: F401

pytestmark = pytest.mark.gpu


def widened(ops, dtype, D):
    return dtype == torch.bfloat16 and D in (64, 128) and ops.prefill_8bit == "tcgen05"


def room(dtype, want, most, portions_from=None):
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
    off = most[..., 0] * 2.0 ** -20 * (most[..., 1] + 8) + 2.0 ** -31 * most[..., 4] * most[..., 3]
    if portions_from is not None:
        off[portions_from:] += most[portions_from:, :, 0] * 2.0 ** -11
    return half * want.abs() + off.repeat_interleave(want.shape[1] // most.shape[1], 1) + 1e-30


def attend(ops, q, H, K, D, pages, ctx, group, scale, window=None, sinks=None):
    out = torch.full((q.shape[0], H * D), 5.0, dtype=q.dtype, device="cuda")
    ops.paged_attention_8bit(q.cuda(), H, K, D, *[t.cuda() for t in pages], plain.cuda(ctx), plain.cuda(group), scale, window, out,
                             sinks=sinks)
    return out.cpu().double()


def check(ops, q, H, K, D, pages, ctx, group, scale, window=None):
    got = attend(ops, q, H, K, D, pages, ctx, group, scale, window)
    want, most = plain.attention(q, H, K, D, *pages, ctx, group, scale, window)
    limit = room(q.dtype, want, most, ctx.n_decode if widened(ops, q.dtype, D) else None)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert bool(((got - want).abs() <= limit).all()), float(((got - want).abs() / limit).max())


# ---- queries of any size -------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("power", [100, 112, 116, 120, -100, -110, -118])
def test_queries_of_any_size(ops, dtype, power):
    """Rows whose largest value is about 2^(power + 2), with a scale that makes ordinary scores of them: what comes out is what
    ordinary rows give.  (The sums of the widened portions are float32's: 2^120 times keys of 4 is as far as they reach.)"""
    for D in (64, 128, 48):
        check_attention(ops, dtype, 4, 2, D, 16, [1, 1, 40], [70, 3, 50], 2, q_scale=2.0 ** power, scale=D ** -0.5 * 2.0 ** -power)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("power", [66, 115, 120, 124])
def test_large_queries_over_small_keys(ops, dtype, power):
    """Sums of whole numbers that a query's power of two would take past float32 before the keys' scale takes them back: scores of
    2^13 and more, of which one is the largest by far.  A score is off by 2^-20 of S, the largest sum |q| |k| scale, at most: where
    the next one is 2^-18 S + 40 behind, each other key weighs e^-39 of the largest at most (which may be lost, being below 2^-31), and the
    result is the largest one's value but for its rounding; where it is nearer, `room` holds."""
    if widened(ops, dtype, 64):
        ops.prefill_8bit = "rows"
    g = torch.Generator().manual_seed(41)
    ctx, group = plain.batch([1, 1, 20], [70, 3, 0], 16, 12, 2)
    k8, _ = pages_of(g, 12, 2, 16, 64)
    v8, vs = pages_of(g, 12, 2, 16, 64)
    ks = torch.full((12, 2), 2.0 ** -60)
    q = rnd(g, 22, 256, scale=2.0 ** power, dtype=dtype)
    got = attend(ops, q, 4, 2, 64, (k8, v8, ks, vs), ctx, group, 0.125)
    want, most = plain.attention(q, 4, 2, 64, k8, v8, ks, vs, ctx, group, 0.125, None)
    limit = room(dtype, want, most, 2 if widened(ops, dtype, 64) else None)
    clear = 0
    for t in range(22):
        r = min(t, 2)
        last = int(ctx.ctx_lens[r]) - (22 - t if r == 2 else 1)
        j = torch.arange(last + 1)
        page = group.block_table[r][j // 16].long()
        for h in range(4):
            s = (k8[page, h // 2, j % 16].double() * 2.0 ** -60) @ q[t, 64 * h:64 * h + 64].double() * 0.125
            two = torch.topk(s, min(2, last + 1)).values
            if last == 0 or float(two[0] - two[1]) >= 2.0 ** -18 * float(most[t, h, 1]) + 40:
                limit[t, 64 * h:64 * h + 64] = 2.0 ** -8 * want[t, 64 * h:64 * h + 64].abs() + (last + 1) * math.exp(-39) * most[t, h, 0]
                clear += 1
    assert clear >= 70
    assert bool(((got - want).abs() <= limit).all())
