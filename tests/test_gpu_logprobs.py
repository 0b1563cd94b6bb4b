"""Log probabilities of given tokens against the same in 64 bits (tests/plain_8bit.py).

Tolerance: the sum of exponentials and its logarithm are off by some 2^-21 of 1 (exponentials of 2^-22, arguments of
2^-23 times up to 20 that weigh e^-20, sums by tree), x - max by 2^-24 of itself, the difference by 2^-24 of the result: 1e-6
and 2^-22 of the result.  The entropy sums p (x - max): 2e-6 and 2^-21 of it."""
import math

import pytest
import torch

import plain_8bit as plain

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from rvllm_b200.kernels import cuda_ops
    return cuda_ops()


def check(ops, x, tokens, top, on=None):
    got = [t.cpu() for t in ops.token_logprobs(x.cuda() if on is None else on, tokens.cuda(), top)]
    assert [t.dtype for t in got] == [torch.float32, torch.int32, torch.float32, torch.float32, torch.int32]
    assert got[3].shape == got[4].shape == (x.shape[0], top)

    def near(a, b, atol, rtol):
        return (math.isnan(a) and math.isnan(b)) or a == b or abs(a - b) <= atol + rtol * abs(b)
    for r, (lp, rank, h, best, ids) in enumerate(plain.logprobs(x, tokens, top)):
        assert near(float(got[0][r]), lp, 1e-6, 2.0 ** -22), (r, float(got[0][r]), lp)
        assert int(got[1][r]) == rank or math.isnan(lp)
        assert near(float(got[2][r]), h, 2e-6, 2.0 ** -21), (r, float(got[2][r]), h)
        assert got[4][r].tolist() == ids, (r, got[4][r].tolist(), ids)
        assert all(near(a, b, 1e-6, 2.0 ** -22) for a, b in zip(got[3][r].tolist(), best))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (1, 2, 0), (3, 7, 7), (2, 33, 32), (5, 1000, 5), (1, 4099, 20), (2, 20001, 32),
                                            (1, 65536, 20), (700, 1031, 3), (1, 131072, 1), (40, 8192, 8)])
def test_rows(ops, dtype, rows, vocab, top):
    g = torch.Generator().manual_seed(vocab)
    x = (torch.randn(rows, vocab, generator=g) * 3).to(dtype)
    tokens = torch.randint(0, vocab, (rows,), generator=g, dtype=torch.int32)
    tokens[0] = int(x[0].argmax())
    if rows > 2:
        tokens[1], tokens[2] = -1, vocab
    check(ops, x, tokens, top)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_orders_and_ties(ops, dtype):
    """Rising and falling rows, all values alike, few different values, the two zeros, the largest at either end."""
    v = 9001
    n = torch.arange(v).float()
    rows = [n / 1000, -n / 1000, torch.full((v,), 2.5), (n * 7919 % 13).floor(), torch.where(n % 2 == 0, 0.0, -0.0),
            torch.where(n == 0, 50.0, 0.0), torch.where(n == v - 1, 50.0, 0.0), (n % 3000) / 100]
    x = torch.stack(rows).to(dtype)
    for top in (1, 8, 9, 32):
        check(ops, x, torch.tensor([0, 1, 4000, 5, 9000, 0, 9000, 2999], dtype=torch.int32), top)


def test_masked_and_not_finite(ops):
    """Logits of -inf, of the type's lowest value, rows of nothing else, NaN, +inf."""
    v = 5000
    g = torch.Generator().manual_seed(3)
    x = torch.randn(9, v, generator=g)
    low = torch.finfo(torch.float32).min
    x[0, 100:] = -math.inf
    x[1, 5:] = -math.inf                                           # fewer left than alternatives
    x[2, 100:] = low
    x[3, :] = low
    x[4, :] = -math.inf
    x[5, 77] = math.nan
    x[6, :] = math.nan
    x[7, 123] = math.inf
    x[8, 3] = -math.inf
    tokens = torch.tensor([5, 2, 200, 7, 9, 4, 1, 123, 3], dtype=torch.int32)
    check(ops, x, tokens, 10)
    check(ops, x.to(torch.bfloat16), tokens, 10)
    check(ops, x, tokens, 0)


def test_strides(ops):
    """Rows of any start and stride, the columns beyond the vocabulary not looked at."""
    g = torch.Generator().manual_seed(4)
    for dtype in (torch.float32, torch.bfloat16):
        wide = (torch.randn(6, 3011, generator=g) * 2).to(dtype)
        wide[:, 2990:] = 99.0
        on = wide.cuda()
        for a in (0, 1, 3, 5):
            for b in (a + 1, a + 6, 2989, 2990):
                check(ops, wide[:, a:b], torch.full((6,), b - a - 1, dtype=torch.int32), min(4, b - a), on=on[:, a:b])


def test_large_logits(ops):
    """Logits far from zero and far apart: differences are taken first."""
    g = torch.Generator().manual_seed(5)
    x = torch.randn(4, 3000, generator=g)
    x[0] += 30000
    x[1] -= 1e6
    x[2] *= 1e30
    x[3] *= 1e-30
    check(ops, x, torch.tensor([1, 2, 3, 4], dtype=torch.int32), 6)


def test_a_row_does_not_depend_on_the_others(ops):
    """The same row alone (eight blocks), among a few and among many (one block): the same largest and ranks; sums within
    their roundings; twice the same call: the same bits."""
    g = torch.Generator().manual_seed(6)
    x = torch.randn(1300, 30011, generator=g).cuda()
    t = torch.randint(0, 30011, (1300,), generator=g, dtype=torch.int32).cuda()
    many = ops.token_logprobs(x, t, 20)
    again = ops.token_logprobs(x, t, 20)
    assert all(torch.equal(a, b) for a, b in zip(many, again))
    for n in (1, 50, 200):
        few = ops.token_logprobs(x[:n], t[:n], 20)
        assert torch.equal(few[1], many[1][:n]) and torch.equal(few[4], many[4][:n])
        for i in (0, 2, 3):
            assert float((few[i] - many[i][:n]).abs().max()) <= 4e-6


def test_no_rows(ops):
    got = ops.token_logprobs(torch.empty(0, 100, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda"), 3)
    assert [tuple(t.shape) for t in got] == [(0,), (0,), (0,), (0, 3), (0, 3)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [4, 900])
def test_tokens_outside_the_vocabulary(ops, dtype, rows):
    """They have rank 0 and no log probability, in rows of any kind; the row's entropy and its largest are what they are."""
    v = 3000
    x = torch.randn(rows, v, generator=torch.Generator().manual_seed(9)).to(dtype)
    x[1, 5] = math.nan
    x[2] = -math.inf
    inside = torch.full((rows,), 7, dtype=torch.int32)
    outside = torch.tensor([-1, v, 2 ** 31 - 1, -2 ** 31] * (rows // 4), dtype=torch.int32)
    a, b = (ops.token_logprobs(x.cuda(), t.cuda(), 3) for t in (inside, outside))
    assert not b[1].any() and torch.isnan(b[0]).all() and bool((a[1] >= 1).all())
    for i in (2, 3, 4):
        assert torch.equal(torch.nan_to_num(a[i], nan=-5.0), torch.nan_to_num(b[i], nan=-5.0))
