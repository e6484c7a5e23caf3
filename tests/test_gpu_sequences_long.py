"""Rows over long caches and prompts, whose parts are added up by several waves, workgroups and launches.  Results are small there (a mean of
many values that cancel): the tolerance (tests/test_gpu_sequences_precision.py) is in proportion to what one row's sums can be off, and that it
notices what is left out is tested for every case, on the CPU."""
import math

import pytest

import fyusenet_amd as fa
from tests.test_gpu_sequences import STORAGE, TYPES, close, stream, visible
from tests.test_gpu_sequences_precision import exact, scores, weighted

torch = pytest.importorskip("torch")

# heads kv dim page, tokens of each sequence before, new tokens, window, sinks
CASES = [
    (2, 1, 64, 16, [40000], 1, 0, 0),                # parts of one row
    (16, 2, 128, 64, [30000, 11111, 7], 1, 0, 0),    # ... of rows of different lengths
    (4, 4, 32, 8, [20000, 1, 9000], 1, 8000, 100),   # a window and first tokens
    (8, 2, 256, 32, [9000, 300], 1, 0, 0),
    (24, 1, 80, 16, [17000], 1, 0, 0),               # more heads of a group than sixteen
    (16, 4, 96, 16, [12000, 5000], 4, 0, 0),         # several new tokens: columns are heads
    (4, 4, 64, 16, [9000, 4000], 20, 0, 0),          # ... columns are tokens
    (4, 4, 128, 32, [9000, 4000], 20, 3000, 40),
    (32, 4, 64, 16, [6000, 3000], 200, 0, 0),        # pieces of a prompt in tiles
    (32, 4, 128, 32, [5000, 3000], 200, 2000, 50),
]


def made(case, typ):
    heads, kv, dim, page, before, new, window, sinks = case
    gen = torch.Generator().manual_seed(dim + new)
    n = [b + new for b in before]
    return [torch.randn(s, generator=gen).to(TYPES[typ]) for s in ((len(n) * new, heads, dim), (sum(n), kv, dim), (sum(n), kv, dim))] + [n]


def rows_of_one(q, heads):
    """Of a piece of many tokens the first and the last ones (a reference of all would take long)."""
    return sorted({0, 1, q.shape[0] // 2, q.shape[0] - 2, q.shape[0] - 1} & set(range(q.shape[0])))


def each(case, typ):
    """(sequence, its rows that are looked at, their position, queries, keys, values)"""
    new = case[5]
    q, k, v, n = made(case, typ)
    at = 0
    for s, m in enumerate(n):
        mine = q[s * new:(s + 1) * new]
        for r in rows_of_one(mine, case[0]):
            yield s, s * new + r, m - new + r, mine[r:r + 1], k[at:at + m], v[at:at + m]
        at += m


def reference(case, pos, q, k, v):
    return exact(q, k, v, pos, k.shape[0] // (8 if case[5] >= 100 else 128) + 100, True, case[6], case[7])


@pytest.mark.parametrize("typ", ["f16", "f32"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "h%d_%d_d%d_p%d_n%d_new%d_w%d_s%d" % (c[:4] + (c[4][0],) + c[5:]))
def test_what_is_left_out_is_noticed(case, typ):
    """Nothing at all, halves, a tenth, a sixteenth, one wave's steps, the first tokens; and parts that are joined without their weights."""
    for s, row, pos, q, k, v in each(case, typ):
        n = k.shape[0]
        if pos < 1000 or pos != n - 1:   # (of each sequence the last row)
            continue
        want, tol = reference(case, pos, q, k, v)
        sc, _ = scores(q.double(), k.double(), pos, True, case[6], case[7], 1 / math.sqrt(case[2]))
        seen = torch.nonzero(visible(torch.tensor([[pos]]), torch.arange(n)[None, :], n, True, case[6], case[7])[0])[:, 0]
        m = len(seen)
        part = {"first half": seen[:m // 2], "second half": seen[m // 2:], "last tenth": seen[-(m // 10):], "all but the last tenth": seen[:-(m // 10)], "a sixteenth": seen[m // 4:m // 4 + m // 16],
                "a wave": seen[(seen // 32) % 4 == 1]}
        if case[7]:
            part["the first tokens"] = seen[:case[7]]
        outs = {"nothing": torch.zeros_like(want)}
        for what, keys in part.items():
            lost = torch.zeros(n, dtype=torch.bool)
            lost[keys] = True
            outs[what] = weighted(sc, v.double(), lost=lost)[0]
        outs["parts joined alike"] = (outs["last tenth"] + outs["all but the last tenth"]) / 2
        for what, got in outs.items():
            assert ((got.to(q.dtype).double() - want).abs() > tol).any(), what
        close(want.to(q.dtype), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("typ", ["f16", "f32"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "h%d_%d_d%d_p%d_n%d_new%d_w%d_s%d" % (c[:4] + (c[4][0],) + c[5:]))
@pytest.mark.parametrize("streams", [1, 3])
def test_long_rows(case, typ, streams):
    """... and with calls that take turns on several streams."""
    heads, kv, dim, page, before, new, window, sinks = case
    q, k, v, n = made(case, typ)
    q, k, v = q.cuda(), k.cuda(), v.cuda()
    count = len(n)
    cache = fa.SequenceCache(STORAGE[typ], 1, heads, kv, dim, page, sum(-(-m // page) for m in n), count)
    first = [sum(n[:s]) for s in range(count)]
    old = torch.cat([torch.arange(f, f + b) for f, b in zip(first, before)]).cuda()
    fresh = torch.cat([torch.arange(f + b, f + m) for f, b, m in zip(first, before, n)]).cuda()
    ko, vo, kf, vf, out = k[old], v[old], k[fresh], v[fresh], torch.full_like(q, math.nan)
    torch.cuda.synchronize()
    use = [torch.cuda.Stream().cuda_stream for _ in range(streams)] if streams > 1 else [stream()]
    who = list(range(count))
    cache.extend(who, before, stream=use[0])
    cache.write(0, ko, vo, stream=use[1 % streams])
    cache.extend(who, [new] * count, stream=use[2 % streams])
    cache.write(0, kf, vf, stream=use[0])
    cache.attend(0, q, out, window=window, sinks=sinks, stream=use[1 % streams])
    cache.order(stream())
    for s, row, pos, a, b, c in each(case, typ):
        close(out[row:row + 1], *reference(case, pos, a, b, c), "sequence %d, row %d" % (s, row))
    torch.cuda.synchronize()


#  batch tokens heads kv dim causal window sinks
PROMPTS = [(1, 6000, 2, 1, 64, True, 0, 0), (1, 6000, 32, 4, 64, True, 0, 0), (1, 4000, 32, 4, 128, False, 0, 0), (1, 9000, 16, 16, 32, True, 3000, 30), (1, 3000, 8, 2, 200, True, 0, 0)]


@pytest.mark.gpu
@pytest.mark.parametrize("typ", ["f16", "f32"])
@pytest.mark.parametrize("case", PROMPTS, ids=lambda c: "t%d_h%d_%d_d%d_%s_w%d_s%d" % (c[1:5] + ("causal" if c[5] else "both",) + c[6:]))
def test_long_prompts(case, typ):
    batch, tokens, heads, kv, dim, causal, window, sinks = case
    gen = torch.Generator().manual_seed(tokens)
    q, k, v = (torch.randn(batch, tokens, h, dim, generator=gen).to(TYPES[typ]).cuda() for h in (heads, kv, kv))
    out = torch.full_like(q, math.nan)
    fa.attention(q, k, v, out, causal=causal, window=window, sinks=sinks, stream=stream())
    assert torch.isfinite(out).all()
    for row in (0, 1, 63, 64, 500, tokens // 2, tokens - 130, tokens - 2, tokens - 1):
        close(out[0, row:row + 1], *exact(q[0, row:row + 1], k[0], v[0], row, tokens // 8 + 100, causal, window, sinks), "row %d" % row)
