"""The cache in 8 bits: its write, pages read back, attention over it, each against the same in 64 bits
(tests/plain_8bit.py), and a layer's step of them together.

Tolerances.  A value held in 8 bits is off by half a step of its page's scale, and where the float32 arithmetic before it
(a norm over `dim` values, a rotation: some 16 roundings of 2^-24 and a sum's) reaches a border between steps by 2^-18 of
its largest value more.  Attention: `plain_8bit.attention_room`."""
import math

import pytest
import torch

import plain_8bit as plain

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16]


@pytest.fixture(params=["blocks-rows", "stream-tcgen05"])
def ops(request):
    """With either kernel for single tokens, and either for the portions that both can take."""
    from rvllm_b200.kernels import cuda_ops
    ops = cuda_ops()
    was = ops.decode_8bit, ops.prefill_8bit
    ops.decode_8bit, ops.prefill_8bit = request.param.split("-")
    yield ops
    ops.decode_8bit, ops.prefill_8bit = was


def rnd(g, *shape, scale=1.0, dtype=torch.float32):
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def angles(positions, dim):
    a = torch.outer(torch.arange(positions, dtype=torch.float64), 10000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim))
    return a.cos().float(), a.sin().float()


def pages_of(g, pages, kv, ps, dim, spread=1.0):
    """Pages as if written: int8 and powers of two."""
    k8 = torch.randint(-127, 128, (pages, kv, ps, dim), generator=g, dtype=torch.int8)
    return k8, 2.0 ** torch.randint(-8, -4, (pages, kv), generator=g).float() * spread


def write_both(ops, rows, H, K, D, qw, kw, eps, table, ctx, group, caches):
    """The call on the GPU and the plain one; caches = (k8, v8, ks, vs) on the host, changed in place."""
    n = rows.shape[0]
    dev = [c.cuda() for c in caches]
    q_out = torch.full((n, H * D), 7.0, dtype=rows.dtype, device="cuda")
    c = lambda t: None if t is None else t.cuda()  # noqa: E731
    ops.qk_norm_rope_write_8bit(rows.cuda(), H, K, D, c(qw), c(kw), eps, None if table is None else tuple(map(c, table)),
                                ctx.positions.cuda(), group.slot_mapping.cuda(), q_out, *dev)
    q, k, v = plain.write(rows, H, K, D, qw, kw, eps, table, ctx.positions, group.slot_mapping, *caches)
    return q_out.cpu(), q, (k, v), [d.cpu() for d in dev]


def check_written(dtype, got_q, q, exact, dev, caches, before):
    step = 2.0 ** -8 if dtype == torch.bfloat16 else 0.0
    assert bool(((got_q.double() - q).abs() <= step * q.abs() + 2.0 ** -18 * q.abs().max()).all())
    for x, cache, scale, want, want_scale, was in ((exact[0], dev[0], dev[2], caches[0], caches[2], before[0]),
                                                   (exact[1], dev[1], dev[3], caches[1], caches[3], before[1])):
        assert torch.equal(scale, want_scale)
        new = ~torch.isnan(x)
        value = cache.double() * scale.double()[:, :, None, None]
        room = scale.double()[:, :, None, None] * (0.5 + 127 * 2.0 ** -18)
        assert bool(((value - x).abs()[new] <= room.expand_as(x)[new]).all())
        assert torch.equal(cache[~new], want[~new])               # others: left, or moved to the larger scale
    assert torch.equal(dev[1], caches[1])                         # values pass no arithmetic


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,K,D,ps,new,old", [
    (4, 2, 64, 16, [1], [0]), (4, 2, 64, 16, [1, 1, 1], [15, 16, 40]), (32, 8, 64, 16, [1] * 5 + [37, 20], [3, 15, 16, 31, 0, 5, 0]),
    (6, 2, 48, 8, [1, 23], [7, 3]), (2, 1, 128, 32, [70, 33], [0, 31]), (3, 3, 80, 5, [12, 9], [2, 0]),
    (2, 2, 256, 64, [1, 130], [63, 5]), (4, 1, 16, 64, [200], [11]), (5, 5, 96, 1, [7], [2]), (2, 1, 32, 7, [50], [3])])
def test_write(ops, dtype, H, K, D, ps, new, old):
    g = torch.Generator().manual_seed(7)
    ctx, group = plain.batch(new, old, ps, 3 + sum(-(-(a + b) // ps) for a, b in zip(new, old)), 0, seed=1)
    n, pages = sum(new), 3 + sum(-(-(a + b) // ps) for a, b in zip(new, old))
    rows = rnd(g, n, (H + 2 * K) * D, dtype=dtype)
    k8, ks = pages_of(g, pages, K, ps, D)
    v8, vs = pages_of(g, pages, K, ps, D, 4.0)
    ks[::3] *= 2.0 ** -6                                           # scales that have to grow
    caches, before = [k8, v8, ks, vs], [k8.clone(), v8.clone()]
    got = write_both(ops, rows, H, K, D, 1 + rnd(g, D, scale=0.1), 1 + rnd(g, D, scale=0.1), 1e-6, angles(300, D), ctx, group, caches)
    check_written(dtype, *got, caches, before)


@pytest.mark.parametrize("norm,turn", [(False, False), (True, False), (False, True)])
def test_write_without_norm_or_rotation(ops, norm, turn):
    g = torch.Generator().manual_seed(8)
    H, K, D, ps = 4, 2, 64, 16
    ctx, group = plain.batch([1, 30], [20, 4], ps, 9, 0)
    k8, ks = pages_of(g, 9, K, ps, D)
    v8, vs = pages_of(g, 9, K, ps, D)
    caches, before = [k8, v8, ks, vs], [k8.clone(), v8.clone()]
    w = 1 + rnd(g, D, scale=0.1) if norm else None
    got = write_both(ops, rnd(g, 31, 8 * D), H, K, D, w, w, 1e-5, angles(64, D) if turn else None, ctx, group, caches)
    check_written(torch.float32, *got, caches, before)


@pytest.mark.parametrize("dtype", DTYPES)
def test_write_of_many_tokens(ops, dtype):
    """As many tokens as take the form for long prompts, pages that begin anywhere in a block's range of tokens, heads that leave
    a warp's lanes without one; values that are not finite, and ones beyond the largest scale, among ordinary ones."""
    g = torch.Generator().manual_seed(19)
    for H, K, D, ps, new, old in ((3, 2, 64, 16, [1, 1, 700, 490, 60], [15, 40, 5, 0, 3]), (1, 1, 48, 64, [1200], [70])):
        pages = 3 + sum(-(-(a + b) // ps) for a, b in zip(new, old))
        ctx, group = plain.batch(new, old, ps, pages, 0, seed=3)
        n = sum(new)
        assert n >= 8 * torch.cuda.get_device_properties(0).multi_processor_count
        rows = rnd(g, n, (H + 2 * K) * D, dtype=dtype)
        finite = rows.clone()
        values = rows[:, (H + K) * D:]
        for t, x in ((3, math.nan), (40, math.inf), (41, -math.inf), (700, math.nan), (900, 3e38), (901, -3e38), (1100, 2.0 ** -70)):
            values[t, (7 * t) % (K * D)] = x
        k8, ks = pages_of(g, pages, K, ps, D)
        v8, vs = pages_of(g, pages, K, ps, D, 4.0)
        caches, before = [k8, v8, ks, vs], [k8.clone(), v8.clone()]
        again = [c.clone() for c in caches]
        w = 1 + rnd(g, D, scale=0.1)
        got = write_both(ops, finite, H, K, D, w, w, 1e-6, angles(1300, D), ctx, group, caches)
        check_written(dtype, *got, caches, before)
        dev = write_both(ops, rows, H, K, D, w, w, 1e-6, angles(1300, D), ctx, group, again)[3]
        assert torch.equal(dev[3], again[3]) and torch.equal(dev[1], again[1])
        assert torch.equal(dev[0], got[3][0]) and torch.equal(dev[2], got[3][2])


def test_write_token_by_token_is_the_portion(ops):
    """A page filled by 16 calls holds what one call leaves, but for the bits that its growing scale dropped: a
    step of the last scale at most in all (halves of steps that double)."""
    g = torch.Generator().manual_seed(9)
    H, K, D, ps = 2, 2, 64, 16
    ctx, group = plain.batch([16], [0], ps, 3, 0)
    rows = rnd(g, 16, 6 * D) * torch.linspace(0.1, 9, 16)[:, None]      # scales that grow all along
    table = tuple(t.cuda() for t in angles(16, D))
    one = [torch.zeros(3, K, ps, D, dtype=torch.int8, device="cuda") for _ in "kv"] + [torch.zeros(3, K, device="cuda") for _ in "kv"]
    many = [t.clone() for t in one]
    q = torch.empty(16, H * D, device="cuda")
    slots, at, dev = group.slot_mapping.cuda(), ctx.positions.cuda(), rows.cuda()
    ops.qk_norm_rope_write_8bit(dev, H, K, D, None, None, 0.0, table, at, slots, q, *one)
    for t in range(16):
        ops.qk_norm_rope_write_8bit(dev[t:t + 1], H, K, D, None, None, 0.0, table, at[t:], slots[t:], q[t:t + 1], *many)
    for i in (0, 1):
        assert torch.equal(one[i + 2], many[i + 2])
        assert int((one[i].int() - many[i].int()).abs().max()) <= 1


def test_write_leaves_what_it_does_not_name(ops):
    """Tokens without a slot (between a page's tokens too), beyond the pages, the same slot twice, rows of another
    stride, a page begun anew over what its last holder left, and all other pages."""
    g = torch.Generator().manual_seed(10)
    H, K, D, ps, pages = 4, 2, 64, 16, 12
    slots = torch.tensor([5 * 16, -1, 5 * 16 + 1, -1, -1, 5 * 16 + 2, 7 * 16 + 9, pages * 16, 2 ** 31 - 1, 3 * 16 + 4, 3 * 16 + 4, -5],
                         dtype=torch.int32)
    n = slots.shape[0]
    ctx, group = plain.batch([1], [0], ps, pages, 0)
    ctx.positions, group.slot_mapping = torch.arange(n, dtype=torch.int32), slots
    wide = rnd(g, n, 8 * D + 24, dtype=torch.bfloat16)
    for rows in (wide[:, :8 * D], wide[:, 3:3 + 8 * D]):
        k8, ks = pages_of(g, pages, K, ps, D)
        v8, vs = pages_of(g, pages, K, ps, D)
        ks[5], vs[5] = math.nan, 2.0 ** 60
        caches, before = [k8, v8, ks, vs], [k8.clone(), v8.clone()]
        dev = [c.cuda() for c in caches]
        q_out = torch.empty(n, H * D, dtype=torch.bfloat16, device="cuda")
        on = wide.cuda()
        view = on[:, :8 * D] if rows.data_ptr() == wide.data_ptr() else on[:, 3:3 + 8 * D]
        ops.qk_norm_rope_write_8bit(view, H, K, D, None, None, 0.0, None, None, slots.cuda(), q_out, *dev)
        q, k, v = plain.write(rows, H, K, D, None, None, 0.0, None, ctx.positions, slots, *caches)
        check_written(torch.bfloat16, q_out.cpu(), q, (k, v), [d.cpu() for d in dev], caches, before)


def test_write_of_what_is_not_finite(ops):
    """NaN is held as 0, infinities as the largest value; neither sets the scale.  Zeros have the smallest
    scale, values of any size one within its range.  A position without an angle shows in the query rows."""
    D, ps = 64, 16
    rows = torch.zeros(6, 3 * D)
    v = rows[:, 2 * D:]
    v[0, :4] = torch.tensor([math.nan, math.inf, -math.inf, 3.0])
    v[2, 0], v[3, 0], v[4, 0] = 3e38, -1e-30, 1e-44
    slots = torch.tensor([0, 16, 32, 48, 64, 80], dtype=torch.int32)
    cache = [torch.zeros(6, 1, ps, D, dtype=torch.int8, device="cuda") for _ in "kv"] + [torch.zeros(6, 1, device="cuda") for _ in "kv"]
    q = torch.empty(6, D, device="cuda")
    table = tuple(t.cuda() for t in angles(4, D))
    at = torch.tensor([0, 1, 2, 3, 4, -1], dtype=torch.int32, device="cuda")
    ops.qk_norm_rope_write_8bit(rows.cuda(), 1, 1, D, None, None, 0.0, table, at, slots.cuda(), q, *cache)
    held, scale = cache[1][:, 0, 0, :4].tolist(), cache[3][:, 0].tolist()
    assert scale == [2.0 ** -5, 2.0 ** -60, 2.0 ** 60, 2.0 ** -60, 2.0 ** -60, 2.0 ** -60]
    assert held[0] == [0, 127, -127, 96] and held[1] == [0] * 4 and held[2][0] == 127 and held[3][0] == 0
    assert torch.isnan(q[4:]).all() and not torch.isnan(q[:4]).any()
    assert not cache[0].any()


@pytest.mark.parametrize("gap", [1, 31, 32, 33, 100])
def test_write_with_gaps(ops, gap):
    """Tokens without a slot between those of one page, before the first one and behind the last, more of them than a warp
    looks at; a page larger than that too."""
    g = torch.Generator().manual_seed(18)
    for ps, dim in ((16, 64), (128, 128)):
        slots = [-1] * gap
        for i in range(ps + 5):
            slots += [3 * ps + i if i < ps else 5 * ps + i - ps] + ([-1] * gap if i in (2, ps - 2, ps + 1) else [])
        slots = torch.tensor(slots + [-1] * gap, dtype=torch.int32)
        n = slots.shape[0]
        k8, ks = pages_of(g, 7, 1, ps, dim)
        v8, vs = pages_of(g, 7, 1, ps, dim)
        caches, before = [k8, v8, ks, vs], [k8.clone(), v8.clone()]
        ctx, group = plain.batch([1], [0], ps, 7, 0)
        ctx.positions, group.slot_mapping = torch.arange(n, dtype=torch.int32) % 90, slots
        got = write_both(ops, rnd(g, n, 4 * dim), 2, 1, dim, None, 1 + rnd(g, dim, scale=0.1), 1e-6, angles(90, dim), ctx, group, caches)
        check_written(torch.float32, *got, caches, before)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K,ps,D", [(2, 16, 64), (1, 5, 48), (3, 64, 256)])
def test_read(ops, dtype, K, ps, D):
    g = torch.Generator().manual_seed(11)
    k8, ks = pages_of(g, 9, K, ps, D)
    ids = torch.tensor([8, 0, 3, 3, -1, 9, 5], dtype=torch.int32)
    got = ops.read_8bit(k8.cuda(), ks.cuda(), ids.cuda(), dtype).cpu()
    want = torch.stack([k8[i].float() * ks[i][:, None, None] if 0 <= i < 9 else torch.zeros(K, ps, D) for i in ids.tolist()])
    assert torch.equal(got.float(), want)
    assert ops.read_8bit(k8.cuda(), ks.cuda(), ids[:0].cuda(), dtype).shape == (0, K, ps, D)


def check_attention(ops, dtype, H, K, D, ps, new, old, n_decode, window=None, sinks=False, scale=None, spread=0.0,
                    spoil=None, stride=0, seed=12, q_scale=1.0):
    g = torch.Generator().manual_seed(seed)
    pages = 2 + sum(-(-max(a + b, 0) // ps) for a, b in zip(new, old))
    ctx, group = plain.batch(new, old, ps, pages, n_decode, seed=seed)
    k8, ks = pages_of(g, pages, K, ps, D)
    v8, vs = pages_of(g, pages, K, ps, D)
    if spread:
        vs = vs * 2.0 ** torch.randint(-int(spread), int(spread) + 1, vs.shape, generator=g).float()
    if spoil:
        spoil(group, ctx, k8, v8, ks, vs)
    n = sum(new)
    wide = rnd(g, n, H * D + stride, scale=q_scale, dtype=dtype)
    q = wide[:, :H * D]
    sink = rnd(g, H) if sinks else None
    scale = D ** -0.5 if scale is None else scale
    out = torch.full((n, H * D), 5.0, dtype=dtype, device="cuda")
    on = wide.cuda()[:, :H * D]
    ops.paged_attention_8bit(on, H, K, D, k8.cuda(), v8.cuda(), ks.cuda(), vs.cuda(), plain.cuda(ctx), plain.cuda(group), scale,
                             window, out, sinks=None if sink is None else sink.cuda())
    want, most = plain.attention(q, H, K, D, k8, v8, ks, vs, ctx, group, scale, window, sink)
    got = out.cpu().double()
    nan = torch.isnan(want)
    tensor = dtype == torch.bfloat16 and D in (64, 128) and stride % D == 0 and ops.prefill_8bit == "tcgen05"
    if tensor:                                                     # what is not valid: of portions, not said how
        assert torch.equal(torch.isnan(got[:n_decode]), nan[:n_decode]) and not torch.isnan(got[~nan]).any()
    else:
        assert torch.equal(torch.isnan(got), nan)
    limit = plain.attention_room(dtype, want, most, n_decode if tensor else None)
    over = ((got - want).abs() > limit) & ~nan
    assert not bool(over.any()), (int(over.sum()), float(((got - want).abs() / limit)[~nan].max()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,K,D,ps", [(4, 1, 64, 16), (8, 8, 64, 16), (32, 8, 64, 8), (12, 1, 64, 32), (40, 2, 64, 64), (16, 2, 128, 16),
                                      (3, 1, 128, 5), (20, 1, 128, 32), (4, 2, 16, 16), (6, 2, 48, 7), (10, 2, 80, 16),
                                      (9, 1, 96, 1), (4, 2, 192, 64), (12, 1, 256, 16)])
def test_single_tokens(ops, dtype, H, K, D, ps):
    new = [1] * 9
    old = [0, 1, 30, 31, 32, 63, 64, 200, 515]
    check_attention(ops, dtype, H, K, D, ps, new, old, 9)
    check_attention(ops, dtype, H, K, D, ps, new, old, 9, window=40, sinks=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,K,D,ps", [(4, 1, 64, 16), (8, 8, 64, 16), (6, 2, 64, 7), (16, 2, 128, 32), (4, 4, 128, 64), (6, 2, 48, 8),
                                      (10, 2, 80, 16), (5, 1, 192, 16), (3, 1, 256, 32), (2, 1, 16, 1)])
def test_portions(ops, dtype, H, K, D, ps):
    check_attention(ops, dtype, H, K, D, ps, [3, 70, 1, 33], [0, 0, 90, 64], 0)
    check_attention(ops, dtype, H, K, D, ps, [1, 1, 40, 17], [64, 9, 130, 0], 2, window=33, sinks=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
def test_portions_of_long_contexts(ops, dtype, D):
    """A few tokens at the end of a long context: several parts a row, put together."""
    check_attention(ops, dtype, 4, 2, D, 16, [5, 150], [1500, 700], 0)
    check_attention(ops, dtype, 4, 1, D, 16, [7], [2100], 0, window=900, sinks=True)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_long_context_of_one(ops, dtype):
    check_attention(ops, dtype, 4, 2, 64, 16, [1], [9000], 1)
    check_attention(ops, dtype, 16, 2, 128, 32, [1, 1], [5000, 3], 2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,share", [(64, 0.5), (64, 0.97), (128, 0.9)])
def test_one_key_beside_many_faint_ones(ops, dtype, D, share):
    """A first key that takes most of the weight, and 9,000 others of some 2^-15 of it and less each, whose values all point
    the same way: what they come to together is in the result."""
    g = torch.Generator().manual_seed(31)
    ctx, group = plain.batch([1, 3], [8999, 8990], 16, 1130, 1)
    k8, ks = pages_of(g, 1130, 1, 16, D)
    k8, ks[:] = k8 // 40, 2.0 ** -7
    v8, vs = pages_of(g, 1130, 1, 16, D)
    v8 = v8.abs() // 2 + 60
    q = rnd(g, 4, D, dtype=dtype)
    for r in (0, 1):
        page = int(group.block_table[r, 0])
        k8[page, 0, 0] = torch.where(q[r].float() > 0, 100, -100).to(torch.int8)
        s = float((k8[page, 0, 0].double() * 2.0 ** -7) @ q[r].double())
        # its score is log(9000 share / (1 - share)), the others' about 0
        scale = math.log(9000 * share / (1 - share)) / s
    out = torch.empty(4, D, dtype=dtype, device="cuda")
    ops.paged_attention_8bit(q.cuda(), 1, 1, D, k8.cuda(), v8.cuda(), ks.cuda(), vs.cuda(), plain.cuda(ctx), plain.cuda(group), scale,
                             None, out)
    want, most = plain.attention(q, 1, 1, D, k8, v8, ks, vs, ctx, group, scale, None)
    assert bool(((out.cpu().double() - want).abs() <= plain.attention_room(dtype, want, most, 1 if ops.prefill_8bit == "tcgen05" else None)).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_requests(ops, dtype):
    """More requests than a warp looks at once, most of them short, some padding."""
    old = [(7 * r) % 50 if r % 5 else -1 for r in range(100)]
    check_attention(ops, dtype, 4, 2, 64, 16, [1] * 100, old, 100)


@pytest.mark.parametrize("dtype", DTYPES)
def test_value_scales_far_apart(ops, dtype):
    """Pages whose values differ by up to 2^40, and scores that leave one key or the whole context."""
    check_attention(ops, dtype, 4, 1, 64, 16, [1, 1, 20], [300, 80, 100], 2, spread=20)
    check_attention(ops, dtype, 4, 1, 64, 16, [1, 1, 20], [300, 80, 100], 2, q_scale=30.0)
    check_attention(ops, dtype, 4, 1, 64, 16, [1, 1, 20], [300, 80, 100], 2, q_scale=1e-20, sinks=True)


def test_rows_behind_the_last_request_stay(ops):
    """Rows of the buffers behind the step's last token are not touched, and no step at all touches none."""
    g = torch.Generator().manual_seed(19)
    for dtype in DTYPES:
        ctx, group = plain.batch([1, 1, 30], [40, 70, 10], 16, 20, 2)
        k8, ks = pages_of(g, 20, 2, 16, 64)
        v8, vs = pages_of(g, 20, 2, 16, 64)
        q = rnd(g, 50, 256, dtype=dtype).cuda()
        out = torch.full((50, 256), 7.0, dtype=dtype, device="cuda")
        pages = [t.cuda() for t in (k8, v8, ks, vs)]
        ops.paged_attention_8bit(q, 4, 2, 64, *pages, plain.cuda(ctx), plain.cuda(group), 0.125, None, out)
        assert bool((out[32:] == 7).all()) and not bool((out[:32] == 7).all(1).any())
        ctx.n_reqs = ctx.n_tokens = ctx.n_decode = 0
        out.fill_(7)
        ops.paged_attention_8bit(q, 4, 2, 64, *pages, plain.cuda(ctx), plain.cuda(group), 0.125, None, out)
        assert bool((out == 7).all())


def test_forms_are_chosen_by_size():
    """Few single tokens take blocks and clusters (one launch), many keys of many requests the stream and its merge."""
    from rvllm_b200.kernels import cuda_ops
    ops = cuda_ops()
    for old, launches in (([700], 1), ([100] * 40, 1), ([3900] * 40, 2), ([60000], 2)):
        ctx, group = plain.batch([1] * len(old), old, 16, 9800, len(old))
        pages = [torch.zeros(9800, 8, 16, 64, dtype=torch.int8, device="cuda") for _ in "kv"] + [torch.ones(9800, 8, device="cuda") for _ in "kv"]
        q = torch.randn(len(old), 2048, device="cuda").bfloat16()
        before = ops.launches
        ops.paged_attention_8bit(q, 32, 8, 64, *pages, plain.cuda(ctx), plain.cuda(group), 0.125, None, torch.empty_like(q))
        assert ops.launches - before == launches, old


def test_more_tokens_than_context(ops):
    """A portion that brings more tokens than its context counts: those before position 0 are zeros."""
    def spoil(group, ctx, k8, v8, ks, vs):
        ctx.ctx_lens[1], ctx.ctx_lens[2] = 3, 1
    for dtype in DTYPES:
        for D in (64, 128):
            check_attention(ops, dtype, 4, 2, D, 16, [1, 40, 200], [5, 0, 30], 1, spoil=spoil)


def test_rows_of_other_strides(ops):
    for dtype in DTYPES:
        for stride in (8, 3, 1):
            check_attention(ops, dtype, 4, 2, 64, 16, [1, 1, 40], [70, 3, 50], 2, stride=stride)


def test_what_is_not_seen_does_not_count(ops):
    """Released pages before a window, slots behind the context, pages of other requests: NaN scales and wild values
    there change nothing; a request without context is zeros; one that may see a key without a page, or whose context is
    longer than its table, is NaN."""
    def spoil(group, ctx, k8, v8, ks, vs):
        used = set()
        for r in range(ctx.n_reqs):
            clen = int(ctx.ctx_lens[r])
            first = max(0, clen - (int(ctx.q_start[r + 1]) - int(ctx.q_start[r])) + 1 - 50) // 16
            group.block_table[r, :first] = -1
            used |= set(group.block_table[r].tolist())
            if clen % 16:
                page = int(group.block_table[r, clen // 16])
                k8[page, :, clen % 16:], v8[page, :, clen % 16:] = 127, -128
        for page in range(k8.shape[0]):
            if page not in used:
                ks[page], vs[page] = math.nan, math.inf
        group.block_table[1] = 10 ** 6                             # no such page
    for dtype in DTYPES:
        for D in (64, 128):
            check_attention(ops, dtype, 4, 2, D, 16, [1, 1, 1, 20, 30, 2], [200, 33, -1, 100, 0, -2], 3, window=50, sinks=True, spoil=spoil)

    def short(group, ctx, k8, v8, ks, vs):
        ctx.ctx_lens[1], ctx.ctx_lens[2] = 10 ** 6, 10 ** 5
    for dtype in DTYPES:
        check_attention(ops, dtype, 4, 2, 64, 16, [1, 1, 20], [200, 33, 100], 2, spoil=short)


def test_nan_in_a_query_stays_in_its_row(ops):
    g = torch.Generator().manual_seed(13)
    ctx, group = plain.batch([1, 1, 30], [40, 70, 10], 16, 20, 2)
    k8, ks = pages_of(g, 20, 2, 16, 64)
    v8, vs = pages_of(g, 20, 2, 16, 64)
    for dtype in DTYPES:
        q = rnd(g, 32, 256, dtype=dtype)
        clean = torch.empty(32, 256, dtype=dtype, device="cuda")
        dirty = clean.clone()
        call = lambda x, o: ops.paged_attention_8bit(x.cuda(), 4, 2, 64, k8.cuda(), v8.cuda(), ks.cuda(), vs.cuda(), plain.cuda(ctx),  # noqa: E731
                                                     plain.cuda(group), 0.125, None, o)
        call(q, clean)
        bad = torch.zeros(32, 4, dtype=torch.bool)
        for t, h, x in ((0, 1, math.nan), (5, 3, math.inf), (31, 0, -math.inf)):
            q[t, h * 64 + 7] = x
            bad[t, h] = True
        call(q, dirty)
        bad = bad.repeat_interleave(64, 1)
        assert torch.isnan(dirty.cpu()[bad]).all()
        assert torch.equal(dirty.cpu()[~bad], clean.cpu()[~bad])


def test_pages_beyond_32_bits(ops):
    """Keys and values more than 2^32 bytes into their tensors, and rows of pages numbered past 2^31 / 2."""
    K, ps, D = 8, 64, 128
    pages = (2 ** 32 + 2 ** 28) // (K * ps * D)
    k8 = torch.zeros(pages, K, ps, D, dtype=torch.int8, device="cuda")
    v8 = torch.zeros_like(k8)
    ks = torch.zeros(pages, K, device="cuda")
    vs = torch.zeros_like(ks)
    g = torch.Generator().manual_seed(14)
    rows = rnd(g, 70, 3 * K * D, dtype=torch.bfloat16)
    at = torch.arange(70, dtype=torch.int32)
    slots = torch.where(at < 64, (pages - 1) * ps + at, (pages - 2) * ps + at - 64).int()
    q = torch.empty(70, K * D, dtype=torch.bfloat16, device="cuda")
    ops.qk_norm_rope_write_8bit(rows.cuda(), K, K, D, None, None, 0.0, None, None, slots.cuda(), q, k8, v8, ks, vs)
    small = [torch.zeros(2, K, ps, D, dtype=torch.int8) for _ in "kv"] + [torch.zeros(2, K) for _ in "kv"]
    plain.write(rows, K, K, D, None, None, 0.0, None, at, torch.where(at < 64, at + ps, at - 64), *small)
    for big, want in zip((k8, v8, ks, vs), small):
        assert torch.equal(big[-2:].cpu(), want)
    assert not k8[:-2].any() and not v8[:-2].any()
    ctx, group = plain.batch([1, 69], [0, 1], ps, 4, 1)
    ctx.ctx_lens[:] = torch.tensor([66, 70])
    group.block_table[:] = torch.tensor([[1, 0], [1, 0]])
    ref, most = plain.attention(rows[:, :K * D], K, K, D, *[s for s in (small[0], small[1], small[2], small[3])], ctx, group, 0.09, None)
    group.block_table[:] = torch.tensor([[pages - 1, pages - 2]] * 2)
    out = torch.empty(70, K * D, dtype=torch.bfloat16, device="cuda")
    ops.paged_attention_8bit(rows.cuda()[:, :K * D], K, K, D, k8, v8, ks, vs, plain.cuda(ctx), plain.cuda(group), 0.09, None, out)
    assert bool(((out.cpu().double() - ref).abs() <= plain.attention_room(torch.bfloat16, ref, most, 1 if ops.prefill_8bit == "tcgen05" else None)).all())


def step_state(seed, dtype, H=8, K=2, D=64, ps=16, new=(1, 1, 1, 30), old=(5, 47, 16, 0)):
    g = torch.Generator().manual_seed(seed)
    pages = 20
    ctx, group = plain.batch(list(new), list(old), ps, pages, 3, seed=3)
    k8, ks = pages_of(g, pages, K, ps, D)
    v8, vs = pages_of(g, pages, K, ps, D)
    rows = rnd(g, sum(new), (H + 2 * K) * D, dtype=dtype)
    return ctx, group, rows, [k8, v8, ks, vs], 1 + rnd(g, D, scale=0.1), angles(128, D)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_step_of_them_together(ops, dtype):
    """Write, then attention over what was written, then log probabilities, as a step does: eagerly, captured and replayed twice
    on new rows, and two captured steps on two streams at once, all against the plain ones."""
    H, K, D = 8, 2, 64
    ctx, group, rows, caches, w, table = step_state(15, dtype)
    c, gr = plain.cuda(ctx), plain.cuda(group)
    head = (torch.randn(900, H * D, generator=torch.Generator().manual_seed(16)) / 16).cuda()
    tokens = torch.arange(rows.shape[0], dtype=torch.int32, device="cuda") * 13

    class Step:
        def __init__(self):
            self.rows, self.cache = rows.cuda().clone(), [t.cuda() for t in caches]
            self.q = torch.empty(rows.shape[0], H * D, dtype=dtype, device="cuda")
            self.out = torch.empty_like(self.q)

        def __call__(self):
            ops.qk_norm_rope_write_8bit(self.rows, H, K, D, w.cuda(), w.cuda(), 1e-6, tuple(t.cuda() for t in table), c.positions,
                                        gr.slot_mapping, self.q, *self.cache)
            ops.paged_attention_8bit(self.q, H, K, D, *self.cache, c, gr, 0.125, None, self.out)
            return ops.token_logprobs(self.out.float() @ head.t(), tokens, 4)

        def run(self, table_c, w_c):
            ops.qk_norm_rope_write_8bit(self.rows, H, K, D, w_c, w_c, 1e-6, table_c, c.positions, gr.slot_mapping, self.q, *self.cache)
            ops.paged_attention_8bit(self.q, H, K, D, *self.cache, c, gr, 0.125, None, self.out)
            return ops.token_logprobs(self.out.float() @ head.t(), tokens, 4)

    eager = Step()
    first = eager()
    host = [t.clone() for t in caches]
    q, _, _ = plain.write(rows, H, K, D, w, w, 1e-6, table, ctx.positions, group.slot_mapping, *host)
    want, most = plain.attention(eager.q.cpu(), H, K, D, *[t.cpu() for t in eager.cache], ctx, group, 0.125, None)
    assert bool(((eager.out.cpu().double() - want).abs() <= plain.attention_room(dtype, want, most, 3 if ops.prefill_8bit == "tcgen05" else None)).all())
    assert all(torch.equal(a.cpu(), b) for a, b in zip(eager.cache[2:], host[2:]))
    # captured: two steps of their own, replayed side by side
    table_c, w_c = tuple(t.cuda() for t in table), w.cuda()
    steps, graphs, outs = [Step(), Step()], [], []
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in steps:
        s.run(table_c, w_c)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(s.run(table_c, w_c))
        graphs.append(graph)
    for trial in range(3):
        for i, s in enumerate(steps):
            s.rows.copy_(rows.cuda() if trial == 0 else rows.cuda().roll(trial + i, 0))
            for t, v in zip(s.cache, caches):
                t.copy_(v)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for i, s in enumerate(steps):
            again = Step()
            again.rows.copy_(s.rows)
            expect = again()
            assert torch.equal(again.out, s.out) and all(torch.equal(a, b) for a, b in zip(expect, outs[i]))
            assert all(torch.equal(a, b) for a, b in zip(again.cache, s.cache))
            if trial == 0:
                assert all(torch.equal(a, b) for a, b in zip(first, outs[i]))


def test_other_streams(ops):
    """Calls on a stream of their own, with what is still being made on another one waited for by the caller."""
    ctx, group, rows, caches, w, table = step_state(17, torch.bfloat16)
    c, gr, t = plain.cuda(ctx), plain.cuda(group), tuple(x.cuda() for x in table)
    results = []
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
        cache = [x.cuda() for x in caches]
        q = torch.empty(rows.shape[0], 512, dtype=torch.bfloat16, device="cuda")
        out = torch.empty_like(q)
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            ops.qk_norm_rope_write_8bit(rows.cuda(), 8, 2, 64, w.cuda(), w.cuda(), 1e-6, t, c.positions, gr.slot_mapping, q, *cache)
            ops.paged_attention_8bit(q, 8, 2, 64, *cache, c, gr, 0.125, 20, out)
        torch.cuda.synchronize()
        results.append(out)
    assert torch.equal(*results)
