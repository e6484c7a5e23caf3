"""Attention over sequences and the paged cache of keys and values, against the formulas in 64 bits.

Tolerance of a result, element by element.  u is half a step of 32 bits (2^-24), U half a step of the storage.
  scores    a sum of dim products in any order and the factors: |error| <= (dim + 4) u |q||k| scale, in units of the exponent
  weights   exp of that, to 4 u (argument and result), and (16-bit storage) at most one rounding to 16 bits, 2^-11
            -> each weight is off by e = (dim + 4) u S + 8 u (1 + R) (+ 2^-11), S the largest |q||k| scale, R the largest
               distance of a score from its maximum that the argument of exp has
  result    a mean of values with these weights, weights' sum and product summed over n keys: 2 e V + 2 n u V, V the largest |v|
            of the sequence, and the final rounding U |result| (and half of the storage's smallest step)
"""
import ctypes
import math
import random

import numpy as np
import pytest

import fyusenet_amd as fa
from fyusenet_amd import capi

torch = pytest.importorskip("torch")

TYPES = {"f16": torch.float16, "f32": torch.float32}
STORAGE = {"f16": fa.STORAGE_F16, "f32": fa.STORAGE_F32}


def stream():
    return torch.cuda.current_stream().cuda_stream


def visible(i, j, n, causal, window, sinks):
    see = j < n
    if causal:
        see = see & (j <= i)
    if window:
        see = see & (((i - j).abs() < window) | (j < sinks))
    return see


def reference(q, k, v, first, causal=True, window=0, sinks=0, scale=0.0):
    """One sequence: q [m, heads, dim] at positions first.., k and v [n, kv_heads, dim] -> result, tolerance (64 bits, CPU)."""
    typ = q.dtype
    q, k, v = (x.detach().cpu().double() for x in (q, k, v))
    m, heads, dim = q.shape
    n = k.shape[0]
    if not m or not n:
        return torch.zeros(m, heads, dim, dtype=torch.float64), torch.zeros(m, heads, dim, dtype=torch.float64)
    k, v = (x.repeat_interleave(heads // x.shape[1], 1) for x in (k, v))
    scale = scale or 1 / math.sqrt(dim)
    see = visible(torch.arange(first, first + m)[:, None], torch.arange(n)[None, :], n, causal, window, sinks)
    s = torch.einsum("mhd,nhd->hmn", q, k) * scale
    s = s.masked_fill(~see, -math.inf)
    top = s.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    out = torch.einsum("hmn,nhd->mhd", p / torch.where(total > 0, total, torch.ones_like(total)), v)
    u, U, tiny = 2.0 ** -24, (2.0 ** -11 if typ == torch.float16 else 2.0 ** -24), (2.0 ** -25 if typ == torch.float16 else 0.0)
    big = float(q.norm(dim=-1).max() * k.norm(dim=-1).max()) * abs(scale)
    e = (dim + 4) * u * big + 8 * u * (1 + 2 * big) + (2.0 ** -11 if typ == torch.float16 else 0.0)
    return out, (2 * e + 2 * n * u) * float(v.abs().max()) * (1 + U) + U * out.abs() + tiny


def close(got, want, tol, what=""):
    off = (got.detach().cpu().double() - want).abs()
    assert torch.isfinite(got).all(), what
    worst = (off - tol).max() if off.numel() else torch.tensor(-1.0)
    assert float(worst) <= 0, "%s: off by %.3g where %.3g is allowed" % (what, float(off.flatten()[(off - tol).argmax()]), float(tol.flatten()[(off - tol).argmax()]))


def values(seed, typ, *shapes):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(s, generator=gen).to(TYPES[typ]).cuda() for s in shapes]


# ---------------------------------------------------------------------------------------------------------------------
# prompts
# ---------------------------------------------------------------------------------------------------------------------
#        batch tokens heads kv dim causal window sinks lengths
PROMPTS = [
    (1, 1, 1, 1, 8, True, 0, 0, None),
    (1, 2, 2, 1, 16, False, 0, 0, None),
    (2, 15, 3, 3, 24, True, 0, 0, [15, 1]),
    (1, 16, 4, 2, 32, False, 3, 0, None),
    (3, 17, 4, 1, 40, True, 5, 2, [17, 0, 9]),
    (1, 33, 2, 2, 64, False, 7, 50, None),
    (2, 64, 8, 2, 64, True, 64, 1, [64, 63]),
    (1, 65, 2, 1, 72, True, 1, 0, None),
    (1, 65, 2, 1, 72, False, 1, 3, None),
    (2, 100, 6, 2, 80, True, 33, 17, [100, 37]),
    (1, 129, 5, 5, 96, False, 0, 0, [128]),
    (2, 197, 12, 12, 64, False, 0, 0, None),
    (1, 257, 4, 2, 128, True, 0, 0, None),
    (1, 300, 4, 2, 128, False, 40, 20, [261]),
    (2, 515, 4, 1, 128, True, 130, 4, [515, 384]),
    (1, 130, 2, 1, 136, True, 0, 0, None),
    (1, 190, 3, 3, 256, True, 70, 5, None),
    (1, 1100, 2, 2, 32, True, 300, 33, None),
    (5, 70, 16, 2, 128, True, 0, 0, [70, 69, 64, 1, 0]),
    # enough heads and sequences for workgroups of 64 queries
    (4, 260, 8, 2, 32, True, 0, 0, None),
    (4, 261, 8, 4, 64, False, 50, 9, [261, 0, 130, 3]),
    (3, 330, 12, 3, 96, True, 100, 70, [330, 65, 64]),
    (2, 290, 16, 4, 128, False, 0, 0, [290, 258]),
    (2, 270, 16, 8, 256, True, 33, 5, None),
    (9, 70, 16, 2, 128, True, 0, 0, [70, 69, 64, 1, 0, 33, 70, 2, 65]),
    # ... and of 128
    (8, 300, 16, 4, 128, True, 0, 0, [300, 299, 257, 256, 128, 127, 1, 0]),
    (8, 270, 16, 2, 32, False, 20, 40, None),
    (8, 290, 16, 16, 64, True, 77, 3, [290, 129, 128, 65, 64, 63, 33, 290]),
    (6, 400, 18, 6, 80, False, 0, 0, [400, 390, 130, 5, 1, 250]),
    (6, 300, 24, 3, 200, True, 150, 140, None),
]


@pytest.mark.gpu
@pytest.mark.parametrize("typ", ["f16", "f32"])
@pytest.mark.parametrize("case", PROMPTS, ids=lambda c: "b%d_t%d_h%d_%d_d%d_%s_w%d_s%d%s" % (c[:5] + ("causal" if c[5] else "both",) + c[6:8] + ("_ragged" if c[8] else "",)))
def test_prompt(case, typ):
    batch, tokens, heads, kv, dim, causal, window, sinks, lengths = case
    q, k, v = values(1 + tokens, typ, (batch, tokens, heads, dim), (batch, tokens, kv, dim), (batch, tokens, kv, dim))
    out = torch.full_like(q, math.nan)
    given = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    fa.attention(q, k, v, out, lengths=given, causal=causal, window=window, sinks=sinks, stream=stream())
    for b in range(batch):
        n = lengths[b] if lengths else tokens
        want, tol = reference(q[b, :n], k[b, :n], v[b, :n], 0, causal, window, sinks)
        close(out[b, :n], want, tol, "sequence %d" % b)
        assert (out[b, n:] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("typ", ["f16", "f32"])
@pytest.mark.parametrize("tokens,heads,dim", [(150, 2, 64), (600, 2, 128), (600, 16, 128), (600, 80, 64)])
def test_prompt_of_values_that_nobody_sees(typ, tokens, heads, dim):
    """NaN and infinities behind a sequence's end, and in tokens that only later rows see."""
    n, bad = tokens - 20, tokens // 2
    q, k, v = values(7, typ, (1, tokens, heads, dim), (1, tokens, 2, dim), (1, tokens, 2, dim))
    lengths = torch.tensor([n], dtype=torch.int32, device="cuda")
    clean = torch.empty_like(q)
    fa.attention(q, k, v, clean, lengths=lengths, window=37, sinks=3, stream=stream())
    want, tol = reference(q[0, :n], k[0, :n], v[0, :n], 0, True, 37, 3)
    close(clean[0, :n], want, tol)
    for x, y in ((math.nan, math.nan), (math.inf, -math.inf), (torch.finfo(TYPES[typ]).min, torch.finfo(TYPES[typ]).max)):
        k2, v2, q2 = k.clone(), v.clone(), q.clone()
        q2[0, n:], k2[0, n:], v2[0, n:] = x, y, x
        k2[0, bad], v2[0, bad] = x, x
        out = torch.full_like(q, 5.0)
        fa.attention(q2, k2, v2, out, lengths=lengths, window=37, sinks=3, stream=stream())
        untouched = torch.ones(n, dtype=torch.bool)
        untouched[bad:min(n, bad + 37)] = False
        assert torch.equal(out[0, :n][untouched.cuda()], clean[0, :n][untouched.cuda()])
        assert (out[0, n:] == 0).all()
        if math.isnan(x):
            assert torch.isnan(out[0, bad:min(n, bad + 37)]).all()
        # infinite values of one head: the rows that see them have them (or NaN, where a weight is too small), no others
        v3 = v.clone()
        v3[0, bad, 1] = math.inf
        fa.attention(q, k, v3, out, lengths=lengths, window=37, sinks=3, stream=stream())
        assert torch.equal(out[0, :n, :heads // 2], clean[0, :n, :heads // 2])
        assert torch.equal(out[0, :n][untouched.cuda()], clean[0, :n][untouched.cuda()])
        assert not torch.isfinite(out[0, bad:min(n, bad + 37), heads // 2:]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("typ", ["f16", "f32"])
def test_prompt_strides_and_scale(typ):
    """Queries, keys and values side by side in one tensor, as one product makes them; heads in front of tokens; a result
    between other columns, which stay as they are."""
    batch, tokens, heads, kv, dim = 2, 77, 4, 2, 48
    both, = values(3, typ, (batch, tokens, heads + 2 * kv, dim))
    q, k, v = both[:, :, :heads], both[:, :, heads:heads + kv], both[:, :, heads + kv:]
    wide = torch.full((batch, tokens, heads, 2 * dim), 9.0, dtype=TYPES[typ], device="cuda")
    fa.attention(q, k, v, wide[..., :dim], causal=False, window=9, sinks=1, scale=0.4, stream=stream())
    for b in range(batch):
        want, tol = reference(q[b], k[b], v[b], 0, False, 9, 1, 0.4)
        close(wide[b, :, :, :dim], want, tol)
    assert (wide[..., dim:] == 9).all()
    ahead = [x.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for x in (q, k, v)]
    out = torch.empty(batch, heads, tokens, dim, dtype=TYPES[typ], device="cuda").permute(0, 2, 1, 3)
    fa.attention(*ahead, out, causal=False, window=9, sinks=1, scale=0.4, stream=stream())
    assert torch.equal(out, wide[..., :dim])


@pytest.mark.gpu
@pytest.mark.parametrize("typ", ["f16", "f32"])
def test_prompt_extremes(typ):
    """Scores that differ by thousands, equal scores, a negative scale; lengths that are out of range."""
    q, k, v = values(4, typ, (1, 90, 1, 64), (1, 90, 1, 64), (1, 90, 1, 64))
    out = torch.empty_like(q)
    for factor, scale in ((30.0, 0.0), (0.0, 0.0), (1.0, -0.7), (4.0, 2.0)):
        fa.attention(q * factor, k * factor, v, out, scale=scale, stream=stream())
        close(out[0], *reference(q[0] * factor, k[0] * factor, v[0], 0, scale=scale), "factor %g" % factor)
    for n in (-5, 1000, -2 ** 31, 2 ** 31 - 1):
        fa.attention(q, k, v, out, lengths=torch.tensor([n], dtype=torch.int32, device="cuda"), stream=stream())
        m = max(0, min(90, n))
        close(out[0, :m], *reference(q[0, :m], k[0, :m], v[0, :m], 0))
        assert (out[0, m:] == 0).all()
    for window, sinks in ((2 ** 31 - 1, 0), (2 ** 31 - 1, 2 ** 31 - 1), (1, 2 ** 31 - 1)):
        for causal in (True, False):
            fa.attention(q, k, v, out, causal=causal, window=window, sinks=sinks, stream=stream())
            close(out[0], *reference(q[0], k[0], v[0], 0, causal, window, sinks))


# ---------------------------------------------------------------------------------------------------------------------
# the cache
# ---------------------------------------------------------------------------------------------------------------------
class Pair:
    """A cache and what it should hold, per sequence and layer, on the GPU."""

    def __init__(self, typ, heads, kv, dim, page, pages, sequences, layers=1, most=0):
        self.cache = fa.SequenceCache(STORAGE[typ], layers, heads, kv, dim, page, pages, sequences, most)
        self.typ, self.heads, self.kv, self.dim, self.layers = typ, heads, kv, dim, layers
        self.k = [[torch.empty(0, kv, dim, dtype=TYPES[typ], device="cuda") for _ in range(layers)] for _ in range(sequences)]
        self.v = [[torch.empty(0, kv, dim, dtype=TYPES[typ], device="cuda") for _ in range(layers)] for _ in range(sequences)]
        self.seed = 100

    def extend(self, who, counts, **sight):
        """New tokens: written, attended to, and looked at."""
        self.cache.extend(who, counts, stream=stream())
        rows = sum(counts)
        for i in range(self.layers):
            self.seed += 1
            k, v, q = values(self.seed, self.typ, (rows, self.kv, self.dim), (rows, self.kv, self.dim), (rows + 3, self.heads, self.dim))
            self.cache.write(i, k, v, stream=stream())
            at = 0
            for s, n in zip(who, counts):
                self.k[s][i], self.v[s][i] = torch.cat([self.k[s][i], k[at:at + n]]), torch.cat([self.v[s][i], v[at:at + n]])
                at += n
            out = torch.full_like(q, 3.0)
            self.cache.attend(i, q[:rows], out[:rows], stream=stream(), **sight)
            at = 0
            for s, n in zip(who, counts):
                total = self.k[s][i].shape[0]
                close(out[at:at + n], *reference(q[at:at + n], self.k[s][i], self.v[s][i], total - n, True, **sight), "sequence %d" % s)
                at += n
            assert (out[rows:] == 3).all()

    def check(self, who=None):
        who = list(range(len(self.k))) if who is None else who
        assert self.cache.lengths(who) == [self.k[s][0].shape[0] for s in who]
        rows = sum(self.cache.lengths(who))
        for i in range(self.layers):
            k, v = (torch.full((rows, self.kv, self.dim), 7.0, dtype=TYPES[self.typ], device="cuda") for _ in range(2))
            self.cache.read(who, i, k, v, stream=stream())
            assert torch.equal(k, torch.cat([self.k[s][i] for s in who])) and torch.equal(v, torch.cat([self.v[s][i] for s in who]))


#       heads kv dim page lengths window sinks
STEPS = [
    (1, 1, 8, 8, [1], 0, 0),
    (4, 2, 32, 16, [1, 2, 16, 17], 0, 0),
    (6, 2, 40, 8, [31, 32, 33, 64], 0, 0),
    (16, 1, 64, 64, [200, 5], 0, 0),
    (40, 2, 64, 32, [130, 129], 0, 0),
    (8, 8, 80, 16, [300, 10, 77], 50, 4),
    (4, 1, 96, 128, [500], 129, 70),
    (8, 2, 128, 16, [1000, 3, 700], 0, 0),
    (8, 2, 128, 1024, [2100], 1, 0),
    (2, 1, 136, 8, [90, 91], 33, 2),
    (4, 2, 256, 32, [400, 33], 0, 0),
    (2, 1, 64, 16, [40000], 0, 0),
    (4, 4, 32, 8, [20000, 1, 9000], 8000, 100),
]


@pytest.mark.gpu
@pytest.mark.parametrize("typ", ["f16", "f32"])
@pytest.mark.parametrize("case", STEPS, ids=lambda c: "h%d_%d_d%d_p%d_n%d_w%d_s%d" % (c[:4] + (max(c[4]),) + c[5:]))
def test_single_tokens_over_the_cache(case, typ):
    heads, kv, dim, page, lengths, window, sinks = case
    p = Pair(typ, heads, kv, dim, page, sum(-(-n // page) for n in lengths) + 2 * len(lengths), len(lengths))
    who = list(range(len(lengths)))
    grown = [(s, n - 1) for s, n in enumerate(lengths) if n > 1]
    for s, n in grown:   # (prompts by themselves are looked at below)
        p.cache.extend([s], [n], stream=stream())
        k, v = values(50 + s, typ, (n, kv, dim), (n, kv, dim))
        p.cache.write(0, k, v, stream=stream())
        p.k[s][0], p.v[s][0] = k, v
    p.extend(who, [1] * len(who), window=window, sinks=sinks)
    p.extend(who[::-1], [1] * len(who), window=window, sinks=sinks)
    p.check()


@pytest.mark.gpu
@pytest.mark.parametrize("typ", ["f16", "f32"])
@pytest.mark.parametrize("heads,kv,dim,page", [(4, 1, 64, 8), (2, 2, 128, 16), (12, 2, 48, 64)])
def test_several_tokens_over_the_cache(typ, heads, kv, dim, page):
    """Prompts in pieces, sequences with one, some and no new tokens in one batch."""
    p = Pair(typ, heads, kv, dim, page, 400, 5, layers=2)
    for counts in ([40, 1, 0, 17, 130], [1, 1, 1, 1, 1], [5, 3, 2, 1, 4], [300, 0, 64, 16, 15], [0, 0, 0, 0, 0], [2, 2, 2, 2, 2]):
        p.extend([3, 0, 4, 1, 2], counts, window=0, sinks=0)
    for counts in ([33, 1, 70], [1, 1, 1], [9, 20, 1]):
        p.extend([1, 2, 0], counts, window=41, sinks=6)
    p.check()


@pytest.mark.gpu
@pytest.mark.parametrize("typ", ["f16", "f32"])
@pytest.mark.parametrize("heads,kv,dim,page,counts", [(16, 4, 64, 8, [260, 3, 257, 100]), (16, 2, 128, 32, [200, 65, 190, 129]), (32, 4, 80, 16, [300, 1, 64, 270, 128, 129])])
def test_pieces_of_prompts_over_the_cache(typ, heads, kv, dim, page, counts):
    """Pieces with enough tokens for tiles, one behind the other."""
    n = len(counts)
    p = Pair(typ, heads, kv, dim, page, 40 * n * 16 // page + 200, n)
    p.extend(list(range(n)), [17 + i for i in range(n)], window=0, sinks=0)
    p.extend(list(range(n))[::-1], counts, window=0, sinks=0)
    p.extend(list(range(n)), counts, window=90, sinks=20)
    p.check()


@pytest.mark.gpu
@pytest.mark.parametrize("typ", ["f16", "f32"])
def test_pages_and_attention_together(typ):
    """What a service does with a cache, step by step: prompts, branches, steps, copies, sequences that are cut and end,
    compaction; every step's attention and all that the cache holds are looked at."""
    p = Pair(typ, 4, 2, 64, 16, 120, 8, layers=2, most=400)
    p.extend([0, 1], [70, 33], window=0, sinks=0)
    p.cache.fork(0, [2, 3, 4], stream=stream())
    for s in (2, 3, 4):
        p.k[s], p.v[s] = list(p.k[0]), list(p.v[0])
    used = p.cache.pages()[0]
    assert used == 5 + 3
    p.check()
    p.extend([2, 0, 3, 4], [1, 1, 1, 1], window=0, sinks=0)       # each takes a page of its own where the shared one is not full
    p.extend([2, 0, 3, 4, 1], [20, 1, 1, 3, 1], window=0, sinks=0)
    p.check()
    p.cache.fork(1, [5], 17, stream=stream())
    p.k[5], p.v[5] = [x[:17] for x in p.k[1]], [x[:17] for x in p.v[1]]
    p.cache.copy([3, 1], [6, 7], stream=stream())
    for a, b in ((3, 6), (1, 7)):
        p.k[b], p.v[b] = list(p.k[a]), list(p.v[a])
    p.check()
    p.extend([5, 6, 7], [1, 2, 40], window=30, sinks=2)
    p.cache.truncate([2, 0], [50, 3], stream=stream())
    for s, n in ((2, 50), (0, 3)):
        p.k[s], p.v[s] = [x[:n] for x in p.k[s]], [x[:n] for x in p.v[s]]
    p.cache.free([4, 3], stream=stream())
    for s in (4, 3):
        p.k[s], p.v[s] = [x[:0] for x in p.k[s]], [x[:0] for x in p.v[s]]
    p.check()
    used, free = p.cache.pages()
    assert p.cache.compact(stream=stream()) == used and p.cache.pages() == (used, free)
    p.check()
    p.extend([0, 1, 2, 3, 5, 6, 7], [1, 1, 1, 90, 1, 1, 1], window=0, sinks=0)
    p.check()
    # more than there is: refused, and nothing has changed
    with pytest.raises(fa.FynException) as e:
        p.cache.extend([1, 2, 3, 5, 6, 7], [400 - n for n in p.cache.lengths([1, 2, 3, 5, 6, 7])], stream=stream())
    assert e.value.code == capi.ERR_STATE
    p.check()


#            heads kv dim page prompt branches
BRANCHES = [
    (8, 2, 64, 16, 1500, 5),
    (6, 1, 48, 8, 1024, 7),
    (4, 4, 128, 64, 2100, 20),
    (16, 2, 256, 32, 1300, 3),
    (24, 2, 96, 16, 1055, 4),
    (20, 1, 40, 8, 1200, 3),      # (more heads of a group than sixteen)
    (2, 1, 128, 16, 1023, 33),    # (pages in common, and fewer tokens than are worth it)
    (8, 4, 32, 128, 9000, 17),
]


@pytest.mark.gpu
@pytest.mark.parametrize("typ", ["f16", "f32"])
@pytest.mark.parametrize("case", BRANCHES, ids=lambda c: "h%d_%d_d%d_p%d_n%d_b%d" % c)
def test_steps_of_branches(case, typ):
    """New tokens of sequences that begin with the same pages: of all, of some, in other orders, with one that is not a branch,
    with one that has grown a long way and one that is cut to what all have."""
    heads, kv, dim, page, prompt, branches = case
    others = list(range(1, branches))
    p = Pair(typ, heads, kv, dim, page, (prompt + 700) // page + 6 * branches + 8, branches + 1)
    p.cache.extend([0], [prompt], stream=stream())
    k, v = values(31, typ, (prompt, kv, dim), (prompt, kv, dim))
    p.cache.write(0, k, v, stream=stream())
    p.cache.fork(0, others[:-1], stream=stream())
    p.cache.fork(0, others[-1:], prompt // page * page, stream=stream())
    for s in range(branches):
        p.k[s][0], p.v[s][0] = (k, v) if s != others[-1] else (k[:prompt // page * page], v[:prompt // page * page])
    everyone = list(range(branches))
    p.extend(everyone, [1] * branches)
    p.extend([1], [600])
    p.extend(everyone[::-1], [1] * branches)
    p.extend([others[-1], 1], [1, 1])
    p.cache.truncate([others[-1]], [prompt // page * page - 3], stream=stream())
    p.k[others[-1]][0], p.v[others[-1]][0] = (x[0][:prompt // page * page - 3] for x in (p.k[others[-1]], p.v[others[-1]]))
    p.extend(everyone, [1] * branches)
    p.extend([branches], [3])
    p.extend(everyone, [1] * branches, window=100, sinks=20)
    p.extend(everyone + [branches], [1] * (branches + 1))
    p.cache.compact(stream=stream())
    p.extend(everyone[1:] + [0], [1] * branches, scale=0.2)
    p.check()


@pytest.mark.gpu
def test_many_sequences_and_pages():
    """More words, rows and moves than one launch's argument holds."""
    n, tokens = 1000, 9
    p = fa.SequenceCache(fa.STORAGE_F16, 1, 2, 1, 8, 8, 2 * n + 1100, n + 1001, 20)
    k, v, q = values(9, "f16", (n * tokens, 1, 8), (n * tokens, 1, 8), (n, 2, 8))
    who = list(range(n))
    p.extend(who, [tokens - 1] * n, stream=stream())
    rows = torch.arange(n * tokens, device="cuda").reshape(n, tokens)
    p.write(0, k[rows[:, :-1].flatten()], v[rows[:, :-1].flatten()], stream=stream())
    p.extend(who, [1] * n, stream=stream())
    p.write(0, k[rows[:, -1]], v[rows[:, -1]], stream=stream())
    out = torch.empty_like(q)
    p.attend(0, q, out, stream=stream())
    for s in (0, 1, 399, 400, 401, 895, 896, 999):
        at = rows[s]
        close(out[s:s + 1], *reference(q[s:s + 1], k[at], v[at], tokens - 1))
    got_k, got_v = torch.empty_like(k), torch.empty_like(v)
    p.read(who, 0, got_k, got_v, stream=stream())
    assert torch.equal(got_k, k) and torch.equal(got_v, v)
    p.fork(3, list(range(n, n + 1001)), stream=stream())
    branch = torch.empty(1001 * tokens, 1, 8, dtype=torch.float16, device="cuda")
    p.read(list(range(n, n + 1001)), 0, branch, branch.clone(), stream=stream())
    assert torch.equal(branch.reshape(1001, tokens, 1, 8), k[rows[3]].expand(1001, tokens, 1, 8))
    p.free(list(range(n, n + 1001)) + who[::2], stream=stream())
    p.copy(who[1::2], who[::2], stream=stream())
    p.free(who[1::2], stream=stream())
    assert p.compact(stream=stream()) == n
    half = torch.empty(n // 2 * tokens, 1, 8, dtype=torch.float16, device="cuda")
    p.read(who[::2], 0, half, half.clone(), stream=stream())
    assert torch.equal(half, k[rows[1::2].flatten()])


@pytest.mark.gpu
def test_lists_around_a_launch():
    """Lists of pages that end a few words in front of and behind the end of one launch's argument, or of two."""
    k, v = values(13, "f16", (2000 * 8, 1, 8), (2000 * 8, 1, 8))
    for pages in list(range(950, 968)) + list(range(1908, 1926)):
        c = fa.SequenceCache(fa.STORAGE_F16, 1, 1, 1, 8, 8, 2010, 3)
        n = pages * 8 - 3
        c.extend([2, 0], [8, n], stream=stream())
        c.write(0, torch.cat([v[:8], k[:n]]), torch.cat([k[:8], v[:n]]), stream=stream())
        got_k, got_v = (torch.empty(n + 8, 1, 8, dtype=torch.float16, device="cuda") for _ in range(2))
        c.read([0, 2], 0, got_k, got_v, stream=stream())
        assert torch.equal(got_k, torch.cat([k[:n], v[:8]])) and torch.equal(got_v, torch.cat([v[:n], k[:8]])), pages


@pytest.mark.gpu
@pytest.mark.parametrize("typ", ["f16", "f32"])
def test_step_of_what_the_cache_does_not_show(typ):
    """NaN in pages behind a sequence's end, in front of its window, and in other sequences' tokens."""
    heads, kv, dim, n = 4, 2, 64, 150
    c = fa.SequenceCache(STORAGE[typ], 1, heads, kv, dim, 16, 40, 2)
    k, v, q = values(21, typ, (n + 30, kv, dim), (n + 30, kv, dim), (1, heads, dim))
    bad = torch.full_like(k, math.nan)
    c.extend([0, 1], [n + 30, n + 30], stream=stream())
    c.write(0, torch.cat([bad, bad]), torch.cat([bad, bad]), stream=stream())   # every page has NaN in it
    c.truncate([0], [0], stream=stream())
    c.extend([0], [n - 1], stream=stream())
    mixed_k, mixed_v = k[:n - 1].clone(), v[:n - 1].clone()
    mixed_k[5:n - 41], mixed_v[5:n - 41] = math.nan, math.inf
    c.write(0, mixed_k, mixed_v, stream=stream())
    c.extend([0], [1], stream=stream())
    c.write(0, k[n - 1:n], v[n - 1:n], stream=stream())
    out = torch.empty_like(q)
    c.attend(0, q, out, window=41, sinks=5, stream=stream())
    close(out, *reference(q, k[:n], v[:n], n - 1, True, 41, 5))


@pytest.mark.gpu
def test_captured_steps():
    """A step captured once and replayed while the sequences grow, with other work in between."""
    heads, kv, dim, layers = 8, 2, 128, 2
    p = Pair("f16", heads, kv, dim, 16, 700, 3, layers, most=3000)
    p.extend([0, 1, 2], [200, 31, 1], window=0, sinks=0)
    k, v, q = values(33, "f16", (layers, 3, kv, dim), (layers, 3, kv, dim), (layers, 3, heads, dim))
    out = torch.empty_like(q)

    def step():
        for i in range(layers):
            p.cache.write(i, k[i], v[i], stream=stream())
            p.cache.attend(i, q[i], out[i], window=0 if i else 90, sinks=0 if i else 3, stream=stream())

    p.cache.extend([0, 1, 2], [1, 1, 1], stream=stream())
    step()
    for s in range(3):
        for i in range(layers):
            p.k[s][i], p.v[s][i] = torch.cat([p.k[s][i], k[i, s:s + 1]]), torch.cat([p.v[s][i], v[i, s:s + 1]])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
        with pytest.raises(fa.FynException) as e:
            p.cache.extend([0], [1], stream=stream())
        assert e.value.code == capi.ERR_STATE
    for turn in range(6):
        if turn == 3:   # long ones from here on
            p.extend([1, 0], [2000, 900], window=0, sinks=0)
            p.cache.compact(stream=stream())
        fresh = values(60 + turn, "f16", k.shape, v.shape, q.shape)
        for a, b in zip((k, v, q), fresh):
            a.copy_(b)
        p.cache.extend([0, 1, 2], [1, 1, 1], stream=stream())
        out.zero_()
        graph.replay()
        for i in range(layers):
            for s in range(3):
                p.k[s][i], p.v[s][i] = torch.cat([p.k[s][i], k[i, s:s + 1]]), torch.cat([p.v[s][i], v[i, s:s + 1]])
                n = p.k[s][i].shape[0]
                close(out[i, s:s + 1], *reference(q[i, s:s + 1], p.k[s][i], p.v[s][i], n - 1, True, 0 if i else 90, 0 if i else 3), "turn %d" % turn)
        torch.cuda.synchronize()
    p.check()


@pytest.mark.gpu
def test_other_streams():
    """Calls on different streams follow each other without the caller's doing."""
    p = Pair("f16", 4, 2, 64, 16, 3000, 2)
    streams = [torch.cuda.Stream() for _ in range(3)] + [torch.cuda.default_stream()]
    torch.cuda.synchronize()
    k, v, q = values(5, "f16", (20000, 2, 64), (20000, 2, 64), (1, 4, 64))
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    p.cache.extend([0], [20000], stream=streams[0].cuda_stream)
    p.cache.write(0, k, v, stream=streams[1].cuda_stream)
    p.cache.copy([0], [1], stream=streams[2].cuda_stream)
    p.cache.truncate([1], [19999], stream=streams[3].cuda_stream)
    p.cache.extend([1], [1], stream=streams[1].cuda_stream)
    p.cache.write(0, k[-1:], v[-1:], stream=streams[0].cuda_stream)
    p.cache.attend(0, q, out, stream=streams[2].cuda_stream)
    p.cache.order(torch.cuda.current_stream().cuda_stream)
    close(out, *reference(q, k, v, 19999))


@pytest.mark.gpu
def test_two_threads():
    """Two caches, each driven by a thread of its own, and attention over tensors in both."""
    import threading
    wrong = []

    def work(seed):
        try:
            own = torch.cuda.Stream()
            with torch.cuda.stream(own):
                p = Pair("f16", 4, 2, 64, 16, 200, 3)
                p.seed = 1000 * seed
                for i in range(6):
                    p.extend([0, 2, 1], [1 + 7 * i * seed, 3, 20], window=0, sinks=0)
                    if i == 2:
                        p.cache.compact(stream=stream())
                q, k, v = values(seed, "f16", (2, 300, 8, 64), (2, 300, 4, 64), (2, 300, 4, 64))
                out = torch.empty_like(q)
                fa.attention(q, k, v, out, stream=stream())
                close(out[1], *reference(q[1], k[1], v[1], 0))
                p.check()
        except BaseException as e:   # noqa: BLE001 -- told to the test's own thread
            wrong.append(e)

    both = [threading.Thread(target=work, args=(s,)) for s in (1, 2)]
    for t in both:
        t.start()
    for t in both:
        t.join()
    assert not wrong, wrong


# ---------------------------------------------------------------------------------------------------------------------
# refusals (no GPU is asked before an argument is)
# ---------------------------------------------------------------------------------------------------------------------
def _attention_desc(**kw):
    d = capi.AttentionDesc()
    d.struct_size = ctypes.sizeof(d)
    d.storage, d.batch, d.tokens, d.heads, d.kv_heads, d.head_dim = capi.STORAGE_F16, 1, 4, 4, 2, 64
    for name, x in kw.items():
        setattr(d, name, x)
    return d


@pytest.mark.parametrize("wrong,code", [
    ({"struct_size": 4}, capi.ERR_INVALID), ({"storage": 2}, capi.ERR_INVALID), ({"heads": 3}, capi.ERR_INVALID), ({"kv_heads": 0}, capi.ERR_INVALID),
    ({"head_dim": 12}, capi.ERR_UNSUPPORTED), ({"head_dim": 264}, capi.ERR_UNSUPPORTED), ({"head_dim": 0}, capi.ERR_UNSUPPORTED),
    ({"window": -1}, capi.ERR_INVALID), ({"sinks": -1}, capi.ERR_INVALID), ({"scale": math.nan}, capi.ERR_INVALID), ({"scale": 3e38}, capi.ERR_INVALID),
    ({"batch": -1}, capi.ERR_INVALID), ({"tokens": -1}, capi.ERR_INVALID), ({"batch": 1 << 20, "tokens": 1 << 20}, capi.ERR_INVALID), ({}, capi.ERR_INVALID),
], ids=lambda x: "_".join("%s%s" % i for i in x.items()) or "null" if isinstance(x, dict) else "")
def test_attention_refuses(wrong, code):
    with pytest.raises(fa.FynException) as e:
        capi.check(capi.lib().fyn_attention(ctypes.byref(_attention_desc(**wrong)), None))
    assert e.value.code == code


def test_attention_of_nothing():
    for wrong in ({"batch": 0}, {"tokens": 0}):
        capi.check(capi.lib().fyn_attention(ctypes.byref(_attention_desc(**wrong)), None))


@pytest.mark.parametrize("wrong,code", [
    ({"struct_size": 4}, capi.ERR_INVALID), ({"storage": 5}, capi.ERR_INVALID), ({"layers": 0}, capi.ERR_INVALID), ({"heads": 5}, capi.ERR_INVALID),
    ({"head_dim": 20}, capi.ERR_UNSUPPORTED), ({"page_tokens": 4}, capi.ERR_UNSUPPORTED), ({"page_tokens": 24}, capi.ERR_UNSUPPORTED),
    ({"page_tokens": 2048}, capi.ERR_UNSUPPORTED), ({"pages": 0}, capi.ERR_INVALID), ({"sequences": 0}, capi.ERR_INVALID), ({"most_tokens": -1}, capi.ERR_INVALID),
    ({"most_tokens": 161}, capi.ERR_INVALID), ({"pages": 1 << 28}, capi.ERR_INVALID), ({"pages": 1 << 20, "sequences": 1 << 20}, capi.ERR_INVALID),
], ids=lambda x: "_".join("%s%s" % i for i in x.items()) if isinstance(x, dict) else "")
def test_cache_refuses_descriptions(wrong, code):
    d = capi.CacheDesc(ctypes.sizeof(capi.CacheDesc), capi.STORAGE_F16, 1, 4, 2, 64, 16, 10, 3, 0)
    for name, x in wrong.items():
        setattr(d, name, x)
    h = ctypes.c_void_p()
    with pytest.raises(fa.FynException) as e:
        capi.check(capi.lib().fyn_cache_create(0, ctypes.byref(d), ctypes.byref(h)))
    assert e.value.code == code and not h.value


def test_null_handles():
    one = (ctypes.c_int32 * 1)(0)
    L, r = capi.lib(), capi.Rows()
    assert L.fyn_cache_destroy(None) == capi.OK
    for rc in (L.fyn_cache_extend(None, 1, one, one, None), L.fyn_cache_write(None, 0, ctypes.byref(r), ctypes.byref(r), 0, None),
               L.fyn_cache_attend(None, 0, ctypes.byref(capi.AttendDesc(ctypes.sizeof(capi.AttendDesc))), None), L.fyn_cache_fork(None, 0, 1, one, -1, None),
               L.fyn_cache_copy(None, 1, one, one, None), L.fyn_cache_truncate(None, 1, one, one, None), L.fyn_cache_free(None, 1, one, None),
               L.fyn_cache_compact(None, None, None), L.fyn_cache_lengths(None, 1, one, one), L.fyn_cache_pages(None, None, None),
               L.fyn_cache_read(None, 1, one, 0, ctypes.byref(r), ctypes.byref(r), 0, None), L.fyn_cache_order(None, None),
               L.fyn_cache_create(0, None, None), L.fyn_attention(None, None)):
        assert rc == capi.ERR_INVALID


def test_python_checks_tensors():
    x = fa.DeviceArray(1 << 20, "float16", (2, 5, 4, 64))
    kv = fa.DeviceArray(1 << 20, "float16", (2, 5, 2, 64))
    for args in ((x, kv, kv, fa.DeviceArray(1 << 20, "float32", (2, 5, 4, 64))), (x, kv, fa.DeviceArray(1 << 20, "float16", (2, 4, 2, 64)), x),
                 (x, kv, kv, fa.DeviceArray(1 << 20, "float16", (2, 5, 4, 64), (5 * 4 * 128, 4 * 128, 128, 2))), (np.zeros(4), kv, kv, x),
                 (torch.zeros(2, 5, 4, 64, dtype=torch.float16), kv, kv, x)):
        with pytest.raises(fa.FynException):
            fa.attention(*args)
    for lengths in (fa.DeviceArray(1 << 20, "int64", (2,)), fa.DeviceArray(1 << 20, "int32", (3,))):
        with pytest.raises(fa.FynException):
            fa.attention(x, kv, kv, x, lengths=lengths)


@pytest.mark.gpu
def test_calls_refuse():
    q, k = values(1, "f16", (1, 8, 4, 64), (1, 8, 2, 64))
    out = torch.full_like(q, 2.0)
    flat = torch.zeros(8 * 4 * 64 + 8, dtype=torch.float16, device="cuda")
    host = torch.zeros(1, 8, 4, 64, dtype=torch.float16).pin_memory()
    odd = torch.zeros(1, 8, 4, 68, dtype=torch.float16, device="cuda")
    for args in ((flat[1:1 + out.numel()].view(1, 8, 4, 64), k, k, out), (q, k, k, odd[..., :64]),
                 (fa.DeviceArray(host.data_ptr(), "float16", host.shape), k, k, out), (fa.DeviceArray(0, "float16", q.shape), k, k, out)):
        with pytest.raises(fa.FynException) as e:
            fa.attention(*args, stream=stream())
        assert e.value.code == capi.ERR_INVALID
    assert (out == 2).all()
    with pytest.raises(fa.FynException):
        fa.attention(q, k, k, out, lengths=fa.DeviceArray(np.zeros(1, np.int32).ctypes.data, "int32", (1,)), stream=stream())
    c = fa.SequenceCache(fa.STORAGE_F16, 2, 4, 2, 64, 16, 4, 3)
    row, kv = q[0], k[0]
    calls = [lambda: c.write(0, kv, kv), lambda: c.attend(0, row, out[0]), lambda: c.extend([3], [1]), lambda: c.extend([0, 0], [1, 1]),
             lambda: c.extend([0], [65]), lambda: c.extend([0], [-1]), lambda: c.extend([0], [1, 2]), lambda: c.fork(0, [0]), lambda: c.fork(0, [1], 1),
             lambda: c.copy([0], [0]), lambda: c.truncate([0], [1]), lambda: c.free([7]), lambda: c.lengths([9]), lambda: c.read([0], 0, kv, kv)]
    for call in calls:
        with pytest.raises(fa.FynException):
            call()
    c.extend([0], [8], stream=stream())
    calls = [lambda: c.write(2, kv, kv), lambda: c.write(-1, kv, kv), lambda: c.write(0, kv[:7], kv[:7]), lambda: c.write(0, kv.float(), kv.float()),
             lambda: c.attend(0, row, out[0], window=-1), lambda: c.attend(0, row[:, :2], out[0]), lambda: c.attend(2, row, out[0]), lambda: c.read([0, 1], 3, kv, kv),
             lambda: c.extend([1, 2], [30, 30])]
    for call in calls:
        with pytest.raises(fa.FynException):
            call()
    assert c.lengths([0, 1, 2]) == [8, 0, 0] and c.pages() == (1, 3)
    c.write(1, kv, kv, stream=stream())
    c.attend(1, row, out[0], stream=stream())
    close(out[0], *reference(row, kv, kv, 0))
    c.close()
    with pytest.raises(fa.FynException):
        c.extend([0], [1])
