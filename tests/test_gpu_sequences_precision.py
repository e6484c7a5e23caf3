"""How exact attention is, against the formula in 64 bits with a tolerance that is in proportion to what is summed up.

u is half a step of 32 bits (2^-24), U half a step of the storage, A the weighted mean of the |values| that a result is the mean of, S the
largest |q||k| scale of a key that the row sees, R <= 2 S the largest distance of a score from its maximum.
  scores   a sum of dim products in any order and the factors: off by at most (dim + 4) u S, in units of the exponent
  weights  exp of that: its argument rounded, u R, its result, 2 u, and the sums' own factors
             32-bit storage  8 u (1 + R) covers them
             16-bit storage  16 u (1 + R): the argument is up to 14 larger, so that weights keep their precision in two 16-bit numbers, which
                             together are off by 2^-22 of the weight and, at most, 2^-31 of the largest one
           -> each weight is off by e, the result by 2 e A, and n 2^-31 V for the smallest weights, V the largest |value|
  sums     of weights and of products, `depth` additions one behind the other at most: 2 depth u A
  result   rounded: U |result|, and half of the storage's smallest step
"""
import math

import pytest

import fyusenet_amd as fa
from tests.test_gpu_sequences import STORAGE, TYPES, close, stream, values, visible

torch = pytest.importorskip("torch")


def scores(q, k, first, causal, window, sinks, scale):
    """Of one sequence in 64 bits on the CPU, [heads, m, n]; what is not seen is -inf.  Also the largest |q||k| scale of a row."""
    m, heads, dim = q.shape
    n = k.shape[0]
    k = k.repeat_interleave(heads // k.shape[1], 1)
    see = visible(torch.arange(first, first + m)[:, None], torch.arange(n)[None, :], n, causal, window, sinks)
    s = torch.einsum("mhd,nhd->hmn", q, k) * scale
    norms = k.norm(dim=-1).t()[:, None, :]
    big = (torch.where(torch.isinf(norms), torch.zeros_like(norms), norms) * see).amax(-1) * q.norm(dim=-1).t() * abs(scale)   # (an infinite score is not rounded)
    return s.masked_fill(~see, -math.inf), big


def weighted(s, v, lost=None, rounded=False):
    """Result and mean of the |values|, [m, heads, dim].  lost: keys that are left out; rounded: weights in 16 bits."""
    v = v.repeat_interleave(s.shape[0] // v.shape[1], 1)
    if lost is not None:
        s = s.masked_fill(lost, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    if rounded:
        p = (p * 64).half().double() / 64
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    return torch.einsum("hmn,nhd->mhd", p, v), torch.einsum("hmn,nhd->mhd", p, v.abs())


def exact(q, k, v, first, depth, causal=True, window=0, sinks=0, scale=0.0):
    """One sequence: q [m, heads, dim] at positions first.., k and v [n, kv_heads, dim] -> result, tolerance (64 bits, CPU)."""
    half = q.dtype == torch.float16
    q, k, v = (x.detach().cpu().double() for x in (q, k, v))
    dim, n = q.shape[2], k.shape[0]
    s, big = scores(q, k, first, causal, window, sinks, scale or 1 / math.sqrt(dim))
    out, mean = weighted(s, v)
    u, U, tiny = 2.0 ** -24, (2.0 ** -11 if half else 2.0 ** -24), (2.0 ** -25 if half else 0.0)
    e = ((dim + 4) * u * big + (16 if half else 8) * u * (1 + 2 * big) + (2.0 ** -22 if half else 0.0)).t()[:, :, None]
    return out, 2 * (e + depth * u) * mean * (1 + U) + (n * 2.0 ** -31 * float(v.abs().max()) if half else 0.0) + U * out.abs() + tiny


#  batch tokens heads kv dim causal window sinks: enough heads and tokens for workgroups of 64 and of 128 queries
WIDE = [
    (4, 260, 16, 2, 32, True, 0, 0), (4, 261, 16, 4, 64, False, 7, 3), (3, 330, 12, 3, 96, True, 100, 70), (2, 290, 32, 4, 128, True, 0, 0), (2, 270, 32, 8, 200, False, 9, 5),
    (8, 300, 24, 4, 32, True, 0, 0), (8, 270, 24, 8, 64, False, 5, 2), (6, 400, 24, 6, 80, True, 0, 0), (8, 290, 24, 8, 128, True, 77, 3), (6, 300, 32, 4, 256, True, 150, 140),
]


def ids(c):
    return "b%d_t%d_h%d_%d_d%d_%s_w%d_s%d" % (c[:5] + ("causal" if c[5] else "both",) + c[6:8])


def wide(case, typ, device):
    """Queries whose scores differ little, so that the weights' own error is what counts."""
    batch, tokens, heads, kv, dim = case[:5]
    gen = torch.Generator().manual_seed(tokens + dim)
    q, k, v = (torch.randn(batch, tokens, n, dim, generator=gen) for n in (heads, kv, kv))
    return [x.to(TYPES[typ]).to(device) for x in (q / 4, k, v)]


@pytest.mark.parametrize("case", WIDE, ids=ids)
def test_rounded_weights_are_noticed(case):
    """The tolerance is no room for weights that are rounded to 16 bits once."""
    q, k, v = wide((1,) + case[1:], "f16", "cpu")
    want, tol = exact(q[0], k[0], v[0], 0, case[1] // 2 + 100, *case[5:])
    s, _ = scores(q[0].double(), k[0].double(), 0, *case[5:], 1 / math.sqrt(case[4]))
    got = weighted(s, v[0].double(), rounded=True)[0].half()
    assert ((got.double() - want).abs() > tol).any()
    close(want.half(), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("typ", ["f16", "f32"])
@pytest.mark.parametrize("case", WIDE, ids=ids)
def test_prompt_keeps_its_weights(case, typ):
    q, k, v = wide(case, typ, "cuda")
    out = torch.full_like(q, math.nan)
    fa.attention(q, k, v, out, causal=case[5], window=case[6], sinks=case[7], stream=stream())
    for b in range(case[0]):
        close(out[b], *exact(q[b], k[b], v[b], 0, case[1] // 2 + 100, *case[5:]), "sequence %d" % b)


# heads kv dim page counts, of new tokens; window sinks: pieces of prompts for workgroups of 64 and of 128 queries
PIECES = [
    (32, 4, 32, 8, [200, 65, 190, 129], 0, 0), (32, 4, 64, 16, [200, 65, 190, 129], 90, 20), (32, 4, 128, 32, [200, 65, 190, 129], 0, 0), (32, 4, 200, 16, [200, 65, 190, 129], 90, 20),
    (48, 6, 32, 16, [300, 1, 64, 270, 128, 129], 90, 20), (48, 6, 64, 64, [300, 1, 64, 270, 128, 129], 0, 0), (48, 6, 128, 16, [300, 1, 64, 270, 128, 129], 90, 20),
    (48, 6, 256, 8, [300, 1, 64, 270, 128, 129], 0, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("typ", ["f16", "f32"])
@pytest.mark.parametrize("case", PIECES, ids=lambda c: "h%d_%d_d%d_p%d_n%d_w%d_s%d" % (c[:4] + (len(c[4]),) + c[5:]))
def test_pieces_over_the_cache_keep_their_weights(case, typ):
    heads, kv, dim, page, counts, window, sinks = case
    n = len(counts)
    cache = fa.SequenceCache(STORAGE[typ], 1, heads, kv, dim, page, sum(-(-(40 + c) // page) for c in counts), n)
    before = [17 + 3 * i for i in range(n)]
    k0, v0, k1, v1, q1 = values(dim, typ, (sum(before), kv, dim), (sum(before), kv, dim), (sum(counts), kv, dim), (sum(counts), kv, dim), (sum(counts), heads, dim))
    q1 = q1 / 4
    cache.extend(list(range(n)), before, stream=stream())
    cache.write(0, k0, v0, stream=stream())
    cache.extend(list(range(n)), counts, stream=stream())
    cache.write(0, k1, v1, stream=stream())
    out = torch.full_like(q1, math.nan)
    cache.attend(0, q1, out, window=window, sinks=sinks, stream=stream())
    a = b = 0
    for old, new in zip(before, counts):
        ks, vs = torch.cat([k0[a:a + old], k1[b:b + new]]), torch.cat([v0[a:a + old], v1[b:b + new]])
        close(out[b:b + new], *exact(q1[b:b + new], ks, vs, old, (old + new) // 2 + 100, True, window, sinks), "sequence at %d" % b)
        a, b = a + old, b + new


# Two weights that differ by a few of the steps that a number of 32 bits near one has, with values 1 and -1: a result that is their difference.
# Of the largest weight's neighbours exp gives 1 - x to a step, 2^-24 there (and may be one step off), so the difference is off by 2 steps at
# most, half of that in the result of two keys; the rest is rounded in proportion.
#   heads tokens batch: sixteen columns, 64 and 128 queries a workgroup
@pytest.mark.gpu
@pytest.mark.parametrize("batch,tokens,heads", [(1, 40, 2), (4, 130, 32), (6, 160, 48)])
@pytest.mark.parametrize("dim", [16, 64, 128])
@pytest.mark.parametrize("later", [0.0, 7.0])
def test_weights_of_32_bits_keep_their_bits(batch, tokens, heads, dim, later):
    """32-bit storage.  later: how much smaller, in powers of two, the weights are that a sequence begins with."""
    first = 33 if later else 0      # (more than one step of keys)
    for steps in (3.3, 5.7, 20.4):
        x = steps * 2.0 ** -24
        q, k, v = (torch.zeros(batch, tokens, n, dim, device="cuda") for n in (heads, 1, 1))
        q[..., 0] = 1
        k[:, :first, 0, 0] = -later * math.log(2)
        k[:, first + 2:, 0, 0] = -80.0
        k[:, first + 1, 0, 0] = -x                          # (exactly: the product with one)
        v[:, first], v[:, first + 1] = 1, -1
        out = torch.empty_like(q)
        fa.attention(q, k, v, out, causal=False, scale=1.0, stream=stream())
        want = -math.expm1(-x) / (1 + math.exp(-x) + first * 2.0 ** -later)
        off = (out.double() - want).abs().max()
        assert float(off) <= 2 * 2.0 ** -24 / (2 + first * 2.0 ** -later) + 2.0 ** -22 * want, "%g steps: off by %.3g of %.3g" % (steps, off, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [16, 64, 136])
def test_weights_of_32_bits_over_the_cache(dim):
    for steps in (3.3, 5.7, 20.4):
        x, n = steps * 2.0 ** -24, 150
        c = fa.SequenceCache(STORAGE["f32"], 1, 4, 2, dim, 16, 10, 1)
        k, v, q = (torch.zeros(m, h, dim, device="cuda") for m, h in ((n, 2), (n, 2), (1, 4)))
        q[..., 0] = 1
        k[..., 0], k[77, :, 0], k[78, :, 0] = -80.0, 0.0, -x
        v[77], v[78] = 1, -1
        c.extend([0], [n - 1], stream=stream())
        c.write(0, k[:-1], v[:-1], stream=stream())
        c.extend([0], [1], stream=stream())
        c.write(0, k[-1:], v[-1:], stream=stream())
        out = torch.empty_like(q)
        c.attend(0, q, out, scale=1.0, stream=stream())
        want = -math.expm1(-x) / (1 + math.exp(-x))
        off = (out.double() - want).abs().max()
        assert float(off) <= 2.0 ** -24 + 2.0 ** -22 * want, "%g steps: off by %.3g of %.3g" % (steps, off, want)
