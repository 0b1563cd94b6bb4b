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


def left_out(q, H, K, D, pages, ctx, group, scale):
    """What a score can be off by because bfloat16 rows are whole numbers of 24 bits, the row's largest value in [2^22, 2^23): the
    rounding of each value, which this repeats, times the keys' size.  A weight is off by as much of itself, the result by twice that
    of the largest value."""
    k8, _, ks, _ = pages
    x = q.double().reshape(q.shape[0], H, D)
    unit = torch.exp2(torch.floor(torch.log2(x.abs().amax(2, keepdim=True))) - 22)
    lost = (torch.round(x / unit) * unit - x).abs()
    off = torch.zeros(q.shape[0], H, dtype=torch.float64)
    for r in range(ctx.n_reqs):
        clen, a, b = int(ctx.ctx_lens[r]), int(ctx.q_start[r]), int(ctx.q_start[r + 1])
        if clen == 0:
            continue
        j = torch.arange(clen)
        page = group.block_table[r][j // group.page_size].long()
        k = (k8[page, :, j % group.page_size].double() * ks[page].double()[..., None]).abs().amax(0)        # [kv, dim]
        off[a:b] = (lost[a:b] * k.repeat_interleave(H // K, 0)).sum(2) * scale
    return off


def attend(ops, q, H, K, D, pages, ctx, group, scale, window=None, sinks=None):
    out = torch.full((q.shape[0], H * D), 5.0, dtype=q.dtype, device="cuda")
    ops.paged_attention_8bit(q.cuda(), H, K, D, *[t.cuda() for t in pages], plain.cuda(ctx), plain.cuda(group), scale, window, out,
                             sinks=sinks)
    return out.cpu().double()


def check(ops, q, H, K, D, pages, ctx, group, scale, window=None):
    got = attend(ops, q, H, K, D, pages, ctx, group, scale, window)
    want, most = plain.attention(q, H, K, D, *pages, ctx, group, scale, window)
    limit = room(q.dtype, want, most, ctx.n_decode if widened(ops, q.dtype, D) else None)
    if q.dtype == torch.bfloat16:
        n = ctx.n_decode if widened(ops, q.dtype, D) else q.shape[0]
        limit[:n] += (2 * most[:n, :, 0] * left_out(q, H, K, D, pages, ctx, group, scale)[:n]).repeat_interleave(D, 1)
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
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("power", [66, 115, 120, 124])
def test_large_queries_over_small_keys(ops, dtype, power, D):
    """Sums of whole numbers that a query's power of two would take past float32 before the keys' scale takes them back: scores of
    2^13 and more, of which one is the largest by far.  A score is off by 2^-20 of S, the largest sum |q| |k| scale, at most: where
    the next one is 2^-18 S + 40 behind, each other key weighs e^-39 of the largest at most (which may be lost, being below 2^-31), and the
    result is the largest one's value but for its rounding; where it is nearer, `room` holds."""
    g = torch.Generator().manual_seed(41)
    ctx, group = plain.batch([1, 1, 20], [70, 3, 0], 16, 12, 2)
    k8, _ = pages_of(g, 12, 2, 16, D)
    v8, vs = pages_of(g, 12, 2, 16, D)
    ks = torch.full((12, 2), 2.0 ** -60)
    q = rnd(g, 22, 4 * D, scale=2.0 ** power, dtype=dtype)
    got = attend(ops, q, 4, 2, D, (k8, v8, ks, vs), ctx, group, 0.125)
    want, most = plain.attention(q, 4, 2, D, k8, v8, ks, vs, ctx, group, 0.125, None)
    limit = room(dtype, want, most, 2 if widened(ops, dtype, D) else None)
    clear = 0
    for t in range(22):
        r = min(t, 2)
        last = int(ctx.ctx_lens[r]) - (22 - t if r == 2 else 1)
        j = torch.arange(last + 1)
        page = group.block_table[r][j // 16].long()
        for h in range(4):
            s = (k8[page, h // 2, j % 16].double() * 2.0 ** -60) @ q[t, D * h:D * h + D].double() * 0.125
            two = torch.topk(s, min(2, last + 1)).values
            if last == 0 or float(two[0] - two[1]) >= 2.0 ** -18 * float(most[t, h, 1]) + 40:
                limit[t, D * h:D * h + D] = 2.0 ** -8 * want[t, D * h:D * h + D].abs() + (last + 1) * math.exp(-39) * most[t, h, 0]
                clear += 1
    assert clear >= 70
    assert bool(((got - want).abs() <= limit).all())


# ---- bits that must not go ------------------------------------------------------------------------------

def opposite_pairs(g, pages, kv, ps, D):
    """Keys 2 i and 2 i + 1 differ by a step in one dimension, their values by their sign: what is left of them shows every bit
    that the weights have."""
    k8, ks = pages_of(g, pages, kv, ps, D)
    v8, vs = pages_of(g, pages, kv, ps, D)
    k8 = k8.clamp(-126, 126)
    k8[:, :, 1::2] = k8[:, :, ::2]
    k8[:, :, 1::2, 5] += 1
    v8[:, :, 1::2] = -v8[:, :, ::2]
    return k8, v8, ks, vs


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,K,D", [(8, 2, 64), (16, 1, 64), (4, 2, 128), (4, 2, 48), (2, 1, 256)])
def test_weights_that_nearly_cancel(ops, dtype, H, K, D):
    g = torch.Generator().manual_seed(42)
    new, old = [1] * 12 + [9, 30], [1, 3, 3, 5, 7, 7, 9, 15, 31, 63, 127, 801, 2, 20]
    pages = sum(-(-(a + b) // 16) for a, b in zip(new, old))
    ctx, group = plain.batch(new, old, 16, pages, 12, seed=4)
    check(ops, rnd(g, sum(new), H * D, dtype=dtype), H, K, D, opposite_pairs(g, pages, K, 16, D), ctx, group, D ** -0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("large", [30.0, 1000.0, 20000.0])
def test_one_large_value_beside_small_ones(ops, dtype, large):
    """A query value that meets zeros takes no bits from the others, on which the scores hang."""
    g = torch.Generator().manual_seed(43)
    for H, K, D in ((8, 2, 64), (4, 1, 128), (6, 2, 48)):
        new, old = [1] * 6 + [25], [1, 7, 15, 100, 333, 900, 40]
        pages = sum(-(-(a + b) // 16) for a, b in zip(new, old))
        ctx, group = plain.batch(new, old, 16, pages, 6, seed=5)
        k8, v8, ks, vs = opposite_pairs(g, pages, K, 16, D)
        k8[..., 3] = 0
        q = rnd(g, sum(new), H * D, dtype=dtype)
        q[:, 3::D] = large
        # (the room counts what is multiplied: the large value meets zeros)
        check(ops, q, H, K, D, (k8, v8, ks, vs), ctx, group, D ** -0.5)


# ---- values of neighbouring pages far apart ---------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("step", [3, 10, 20, 30])
def test_pages_side_by_side_far_apart(ops, dtype, D, step):
    """Values that grow by 2^step from a page of eight tokens to the next, and that fall so: rows see the first pages alone, or all
    of them, and what a row sees is right by its own largest value."""
    g = torch.Generator().manual_seed(44)
    for sign in (1, -1):
        ctx, group = plain.batch([1, 32, 70], [31, 0, 40], 8, 24, 1, seed=6)
        k8, ks = pages_of(g, 24, 2, 8, D)
        v8, vs = pages_of(g, 24, 2, 8, D)
        for r in range(3):
            for b, page in enumerate(group.block_table[r].tolist()):
                if page >= 0:
                    vs[page] = 2.0 ** max(-60, min(60, sign * (step * (b % 4) - 45)))
        check(ops, rnd(g, 103, 4 * D, dtype=dtype), 4, 2, D, (k8, v8, ks, vs), ctx, group, D ** -0.5)
        sinks = rnd(g, 4)
        got = attend(ops, (q := rnd(g, 103, 4 * D, dtype=dtype)), 4, 2, D, (k8, v8, ks, vs), ctx, group, D ** -0.5, 20, sinks.cuda())
        want, most = plain.attention(q, 4, 2, D, k8, v8, ks, vs, ctx, group, D ** -0.5, 20, sinks)
        assert bool(((got - want).abs() <= room(dtype, want, most, 1 if widened(ops, dtype, D) else None)).all())


@pytest.mark.parametrize("D", [64, 128])
def test_portions_of_long_contexts_far_apart(ops, D):
    """The same where the tiles of a portion are shared out over blocks and put together."""
    g = torch.Generator().manual_seed(45)
    new, old = [40, 5], [2000, 700]
    pages = sum(-(-(a + b) // 16) for a, b in zip(new, old))
    ctx, group = plain.batch(new, old, 16, pages, 0, seed=7)
    k8, ks = pages_of(g, pages, 1, 16, D)
    v8, vs = pages_of(g, pages, 1, 16, D)
    vs = vs * 2.0 ** torch.randint(-9, 9, vs.shape, generator=g).float()
    vs[::7] *= 2.0 ** -30
    check(ops, rnd(g, 45, 4 * D, dtype=torch.bfloat16), 4, 1, D, (k8, v8, ks, vs), ctx, group, D ** -0.5)


def test_the_same_call_gives_the_same_bits(ops):
    g = torch.Generator().manual_seed(46)
    for dtype in DTYPES:
        for D in (64, 128):
            new, old = [1] * 20 + [60, 300], [97 * i + 5 for i in range(20)] + [900, 0]
            pages = sum(-(-(a + b) // 16) for a, b in zip(new, old))
            ctx, group = plain.batch(new, old, 16, pages, 20, seed=8)
            k8, ks = pages_of(g, pages, 2, 16, D)
            v8, vs = pages_of(g, pages, 2, 16, D)
            q = rnd(g, sum(new), 8 * D, dtype=dtype)
            first = attend(ops, q, 8, 2, D, (k8, v8, ks, vs), ctx, group, D ** -0.5)
            for _ in range(3):
                assert torch.equal(first, attend(ops, q, 8, 2, D, (k8, v8, ks, vs), ctx, group, D ** -0.5))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,K,D", [(2, 2, 64), (4, 2, 64), (3, 1, 64), (4, 1, 128), (2, 2, 48), (5, 1, 64), (8, 8, 256)])
def test_portions_of_a_few_rows(ops, dtype, H, K, D):
    """Portions of two to four tokens alone: four rows and fewer a key/value head, and just more."""
    g = torch.Generator().manual_seed(51)
    for new, old in (([2, 2], [0, 30]), ([2, 3, 4], [100, 0, 700]), ([1, 2, 1], [40, 5, 9]), ([4] * 40, [13 * i for i in range(40)])):
        pages = sum(-(-(a + b) // 16) for a, b in zip(new, old))
        new, old = zip(*sorted(zip(new, old), key=lambda e: e[0] != 1))
        ctx, group = plain.batch(list(new), list(old), 16, pages, sum(n == 1 for n in new), seed=10)
        pages_ = opposite_pairs(g, pages, K, 16, D)
        for window in (None, 3):
            check(ops, rnd(g, sum(new), H * D, dtype=dtype), H, K, D, pages_, ctx, group, D ** -0.5, window)


@pytest.mark.parametrize("D", [64, 128])
def test_portions_widened_in_passes(ops, D, monkeypatch):
    """Portions of which memory holds one or two at a time, beside single tokens and an empty one, and the same call captured."""
    g = torch.Generator().manual_seed(47)
    new, old = [1, 1, 40, 70, 3, 0, 130], [30, 200, 500, 0, 90, -1, 300]
    pages = sum(-(-max(0, a + b) // 16) for a, b in zip(new, old))
    ctx, group = plain.batch(new, old, 16, pages, 2, seed=9)
    k8, ks = pages_of(g, pages, 2, 16, D)
    v8, vs = pages_of(g, pages, 2, 16, D)
    q = rnd(g, sum(new), 4 * D, dtype=torch.bfloat16)
    for window in (None, 60):
        a_portion = 4 * 2 * D * (min(ctx.max_ctx_len, window + ctx.max_q_len) if window else ctx.max_ctx_len)
        for n in (1, 2, 5):
            monkeypatch.setattr(ops, "widen_8bit_bytes", n * a_portion)
            check(ops, q, 4, 2, D, (k8, v8, ks, vs), ctx, group, D ** -0.5, window)
    monkeypatch.setattr(ops, "widen_8bit_bytes", 2 * a_portion)
    dev, on, out = [plain.cuda(ctx), plain.cuda(group)], [t.cuda() for t in (k8, v8, ks, vs)], torch.empty_like(q).cuda()
    call = lambda: ops.paged_attention_8bit(q_dev, 4, 2, D, *on, *dev, D ** -0.5, 60, out)  # noqa: E731
    q_dev = q.cuda()
    call()
    torch.cuda.synchronize()
    want = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


# ---- keys that lie beside a border -----------------------------------------------------------------------

@pytest.mark.parametrize("n", [16, 1300])
def test_keys_beside_a_border(ops, n):
    """Keys half way between two steps but for 2^-30 of a turn, and largest values that pass 127 steps by as much: what a page holds
    is the value's own rounding, not that of its rounding to float32, scales included."""
    ps, D = 16, 64
    g = torch.Generator().manual_seed(49)
    ctx, group = plain.batch([n], [0], ps, -(-n // ps) + 1, 0)
    rows = torch.zeros(n, 3 * D)
    k = rows[:, D:2 * D]
    k[:, :D // 2] = (torch.randint(-126, 126, (n, D // 2), generator=g) + 0.5) * 2.0 ** -5
    k[:, D // 2:] = torch.where(torch.rand(n, D // 2, generator=g) < 0.5, -1.0, 1.0)
    k[::3, 0] = torch.where(torch.rand(k[::3, 0].shape, generator=g) < 0.5, -127.0, 127.0) * 2.0 ** -5
    k[5::ps, 1] = 127 * 2.0 ** -5
    table = torch.ones(n, D // 2), torch.full((n, D // 2), 2.0 ** -30)
    pages = group.block_table.shape[1] + 1
    host = [torch.zeros(pages, 1, ps, D, dtype=torch.int8) for _ in "kv"] + [torch.ones(pages, 1) for _ in "kv"]
    dev = [t.cuda() for t in host]
    ops.qk_norm_rope_write_8bit(rows.cuda(), 1, 1, D, None, None, 0.0, tuple(t.cuda() for t in table), ctx.positions.cuda(),
                                group.slot_mapping.cuda(), torch.empty(n, D, device="cuda"), *dev)
    plain.write(rows, 1, 1, D, None, None, 0.0, table, ctx.positions, group.slot_mapping, *host)
    assert torch.equal(dev[2].cpu(), host[2])
    assert torch.equal(dev[0].cpu(), host[0]), int((dev[0].cpu() != host[0]).sum())


@pytest.mark.parametrize("dtype", DTYPES)
def test_keys_are_the_formulas(ops, dtype):
    """Two million keys, normed and turned: every one the rounding of what 64 bits give."""
    n, K, D, ps = 4000, 8, 64, 16
    g = torch.Generator().manual_seed(50)
    rows = rnd(g, n, 3 * K * D, dtype=dtype).cuda()
    w = (1 + rnd(g, D, scale=0.1)).cuda()
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    angle = torch.outer(torch.arange(n, dtype=torch.float64), 1e4 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D))
    cos, sin = angle.cos().float().cuda(), angle.sin().float().cuda()
    pages = [torch.zeros(n // ps, K, ps, D, dtype=torch.int8, device="cuda") for _ in "kv"] + [torch.ones(n // ps, K, device="cuda") for _ in "kv"]
    ops.qk_norm_rope_write_8bit(rows, K, K, D, w, w, 1e-5, (cos, sin), pos, pos, torch.empty(n, K * D, dtype=dtype, device="cuda"), *pages)
    x = rows[:, K * D:2 * K * D].double().view(n, K, D)
    x = x / torch.sqrt((x * x).mean(2, keepdim=True) + 1e-5) * w.double()
    a, b = x.chunk(2, 2)
    c, s = cos.double()[:, None], sin.double()[:, None]
    x = torch.cat([a * c - b * s, a * s + b * c], 2).view(n // ps, ps, K, D).transpose(1, 2)
    most = x.abs().amax((2, 3))
    scale = torch.exp2(torch.ceil(torch.log2(most / 127)))
    scale = torch.where(most > 127 * scale, 2 * scale, torch.where(most <= 63.5 * scale, scale / 2, scale))
    assert torch.equal(pages[2].double(), scale)
    want = torch.round(x / scale[:, :, None, None])
    assert torch.equal(pages[0].double(), want), int((pages[0].double() != want).sum())
