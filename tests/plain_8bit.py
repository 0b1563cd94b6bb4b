"""The 8-bit cache and the log probabilities in 64 bits, written out one token, page and row at a time."""
import math
from types import SimpleNamespace

import torch


def turned(x, w, eps, cos, sin):
    """A head [dim] in float64: RMS norm (w None: none), then the halves turned by the angles (cos None: not)."""
    if w is not None:
        x = x / math.sqrt(float((x * x).mean()) + eps) * w
    if cos is not None:
        h = x.shape[0] // 2
        x = torch.cat([x[:h] * cos - x[h:] * sin, x[:h] * sin + x[h:] * cos])
    return x


def scale_for(x):
    """The smallest power of two s in [2^-60, 2^60] with max |x| <= 127 s over the finite x."""
    x = x[torch.isfinite(x)].abs()
    most = float(x.max()) if x.numel() else 0.0
    e = -60
    while e < 60 and most > 127 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def write(rows, heads, kv, dim, qw, kw, eps, table, positions, slots, k8, v8, ks, vs):
    """What `qk_norm_rope_write_8bit` does.  Returns (q float64 [tokens, heads * dim], the exact values that were put
    into k8 and v8: float64 of their shape, NaN where nothing was written).  k8, v8, ks, vs (host) are changed."""
    n, (pages, _, ps, _) = rows.shape[0], k8.shape
    x = rows[:, :(heads + 2 * kv) * dim].double().reshape(n, heads + 2 * kv, dim)
    angle = lambda t: (None, None) if table is None else (table[0][positions[t]].double(), table[1][positions[t]].double())  # noqa: E731
    w = lambda v: None if v is None else v.double()  # noqa: E731
    q = torch.stack([torch.cat([turned(x[t, h], w(qw), eps, *angle(t)) for h in range(heads)]) for t in range(n)])
    by_page = {}
    for t in range(n):
        s = int(slots[t])
        if 0 <= s < pages * ps:
            by_page.setdefault(s // ps, {})[s % ps] = t            # of two tokens the later one
    put = []
    for first, weight, turn, cache, scale in ((heads, w(kw), True, k8, ks), (heads + kv, None, False, v8, vs)):
        exact = torch.full(cache.shape, math.nan, dtype=torch.float64)
        for page, at in by_page.items():
            for g in range(kv):
                new = {s: (turned(x[t, first + g], weight, eps, *(angle(t) if turn else (None, None))))
                       for s, t in at.items()}
                need = scale_for(torch.stack(list(new.values())))
                if 0 not in at:
                    old = float(scale[page, g])
                    need = max(need, old)
                    if need != old:
                        cache[page, g] = torch.round(cache[page, g].double() * (old / need)).to(torch.int8)
                scale[page, g] = need
                for s, v in new.items():
                    exact[page, g, s] = v
                    cache[page, g, s] = torch.nan_to_num(v / need, nan=0.0, posinf=127, neginf=-127).round().clamp(-127, 127).to(torch.int8)
        put.append(exact)
    return q, put[0], put[1]


def batch(new, old, ps, pages, n_decode, seed=0, width=None, pad_tokens=0):
    """Step arrays of requests with `new` tokens after `old` ones, pages in random order.  On the host; `cuda` moves them.  A
    request with old < 0 is padding: no context."""
    g = torch.Generator().manual_seed(seed)
    lens = [0 if b < 0 else a + b for a, b in zip(new, old)]
    blocks = [-(-n // ps) for n in lens]
    width = width or max(blocks + [1])
    order = torch.randperm(pages, generator=g)
    assert sum(blocks) <= pages
    table, at = torch.full((len(new), width), -1, dtype=torch.int32), 0
    for r, n in enumerate(blocks):
        table[r, :n] = order[at:at + n].int()
        at += n
    slots, positions, req = [], [], []
    for r, (a, b) in enumerate(zip(new, old)):
        for i in range(a):
            p = max(b, 0) + i
            positions.append(p)
            req.append(r)
            slots.append(int(table[r, p // ps]) * ps + p % ps if b >= 0 else -1)
    slots += [-1] * pad_tokens
    positions += [0] * pad_tokens
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    q_start = i32([sum(new[:r]) for r in range(len(new) + 1)])
    ctx = SimpleNamespace(n_reqs=len(new), n_tokens=len(req), n_decode=n_decode, q_start=q_start, ctx_lens=i32(lens),
                          positions=i32(positions), token_req=i32(req), max_q_len=max(new + [1]), max_ctx_len=max(lens + [1]))
    group = SimpleNamespace(block_table=table, slot_mapping=i32(slots), max_blocks=width, page_size=ps, window=None)
    return ctx, group


def cuda(o):
    return SimpleNamespace(**{k: v.cuda() if torch.is_tensor(v) else v for k, v in vars(o).items()})


def attention(q, heads, kv, dim, k8, v8, ks, vs, ctx, group, scale, window, sinks=None):
    """float64 [tokens, heads * dim], and per token and head what its roundings are measured by: the largest |v| seen, the
    largest sum |q| |k| scale, max |q| times the largest norm of a key times scale, the largest weight times 127 times
    its value's scale, and the root of the number of keys."""
    G, ps = heads // kv, group.page_size
    n = q.shape[0]
    out = torch.zeros(n, heads * dim, dtype=torch.float64)
    most = torch.zeros(n, heads, 5, dtype=torch.float64)
    for r in range(ctx.n_reqs):
        clen, a, b = int(ctx.ctx_lens[r]), int(ctx.q_start[r]), int(ctx.q_start[r + 1])
        if clen == 0 or a == b:
            continue
        if clen > group.block_table.shape[1] * ps:
            out[a:b] = math.nan
            continue
        j = torch.arange(clen)
        page = group.block_table[r][j // ps].long()
        there = (page >= 0) & (page < k8.shape[0])
        p0 = page.clamp(0, k8.shape[0] - 1)
        k = k8[p0, :, j % ps].double() * ks[p0].double()[..., None]              # [keys, kv, dim]
        v = v8[p0, :, j % ps].double() * vs[p0].double()[..., None]
        for t in range(a, b):
            p = clen - (b - a) + (t - a)
            seen = j <= p
            if window:
                seen &= j > p - window
            if not bool(seen.any()):
                continue
            if bool((seen & ~there).any()):                       # a visible key without a page
                out[t] = math.nan
                continue
            for h in range(heads):
                x = q[t, h * dim:(h + 1) * dim].double()
                kk, vv = k[seen, h // G], v[seen, h // G]
                s = kk @ x * scale
                if sinks is not None:
                    s = torch.cat([s, sinks[h:h + 1].double()])
                w = torch.softmax(s, 0)[:kk.shape[0]]
                out[t, h * dim:(h + 1) * dim] = w @ vv
                most[t, h, 0] = vv.abs().max()
                most[t, h, 1] = (kk.abs() @ x.abs()).max() * scale
                most[t, h, 2] = x.abs().max() * kk.norm(dim=1).max() * scale
                most[t, h, 3] = (w * vs[p0][seen, h // G].double()).max() * 127
                most[t, h, 4] = math.sqrt(kk.shape[0])
    return out, most


def logprobs(x, tokens, top):
    """Per row: (log p of the token, rank, entropy, the largest logits' log p, their ids), lists of float64 and int."""
    out = []
    for row, t in zip(x.double(), tokens.tolist()):
        # the largest is taken away first: log sum exp itself would lose 9 beside a lowest value of -3e38
        away = row - row.max()
        lse = torch.logsumexp(away, 0)
        lp = away - lse
        p = lp.exp()
        known = 0 <= t < row.shape[0]
        h = -(torch.where(p > 0, p * lp, torch.zeros_like(p))).sum() if bool(torch.isfinite(lse)) else lse * math.nan
        order = sorted((i for i in range(row.shape[0]) if not math.isnan(row[i])), key=lambda i: (-float(row[i]), i))[:top]
        out.append((float(lp[t]) if known else math.nan, int((row > row[t]).sum()) + 1 if known else 0, float(h),
                    [float(lp[i]) for i in order] + [math.nan] * (top - len(order)), order + [-1] * (top - len(order))))
    return out


def attention_room(dtype, want, most, first_portion=None):
    """How far attention may be off, per element.

    float32: the result's rounding (2^-24); weights and scores from float32 sums, operands of 22 bits and exponentials of 2^-22: 2^-20
    of the largest value seen for each unit of the largest sum |q| |k| scale, and 8 units of them.  bfloat16: the result's
    rounding (2^-8), the same, weights rounded to float16 (half a step is 2^-11 of itself: as much of the largest value;
    below 2^-14 of at most 2^6 steps are 2^-24: 2^-31 sqrt(keys) of the largest term), and queries as whole numbers of 16
    bits, in steps of 2^-14 of a row's largest at most: over a key's dimensions a score off by 6 * 2^-14 / sqrt(12) max
    |q| |k| scale (six standard deviations), a weight by as much of itself, the result by twice that of the largest value.
    Tokens from `first_portion` on: weights rounded to bfloat16 (half a step is 2^-8 of itself), queries as they are."""
    dim = want.shape[1] // most.shape[1]
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
    room = most[..., 0] * 2.0 ** -20 * (most[..., 1] + 8)
    if dtype == torch.bfloat16:
        n = want.shape[0] if first_portion is None else first_portion
        whole = most[..., 0] * (2.0 ** -11 + 2 * 6 / math.sqrt(12) * 2.0 ** -14 * most[..., 2]) + 2.0 ** -31 * most[..., 4] * most[..., 3]
        room[:n] += whole[:n]
        room[n:] += most[n:, :, 0] * 2.0 ** -8
    return half * want.abs() + room.repeat_interleave(dim, 1) + 1e-30
