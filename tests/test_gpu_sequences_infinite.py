"""Keys and values that are infinite and seen: a score of minus infinity is a weight of zero, whatever the size of a head, and an infinite value
that weighs something makes an infinite result.  Tolerances: tests/test_gpu_sequences_precision.py."""
import math

import pytest

import fyusenet_amd as fa
from tests.test_gpu_sequences import STORAGE, TYPES, close, stream, values, visible
from tests.test_gpu_sequences_precision import exact

torch = pytest.importorskip("torch")

SIZES = [(1, 75, 2), (4, 130, 32), (6, 160, 48)]   # sixteen columns, 64 and 128 queries a workgroup
DIMS = [8, 16, 24, 32, 40, 48, 56, 64, 72, 80, 88, 96, 104, 112, 120, 128, 136, 184, 200, 248, 256]


def infinite_keys(k, q, where):
    """Minus infinity in the last value, or in the first, of the keys at `where`, for queries that are positive there: their scores are minus infinity."""
    k = k.clone()
    q[..., -1], q[..., 0] = 1 + q[..., -1].abs(), 1 + q[..., 0].abs()
    for i, j in enumerate(where):
        k[..., j, :, -1 if i % 2 == 0 else 0] = -math.inf
    return k


@pytest.mark.gpu
@pytest.mark.parametrize("typ", ["f16", "f32"])
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("batch,tokens,heads", SIZES)
def test_prompt_with_infinite_keys(typ, dim, batch, tokens, heads):
    q, k, v = values(dim, typ, (batch, tokens, heads, dim), (batch, tokens, 2, dim), (batch, tokens, 2, dim))
    k = infinite_keys(k, q, (3, 40, 41, 64, 70))
    for causal, window in ((True, 0), (False, 50)):
        out = torch.empty_like(q)
        fa.attention(q, k, v, out, causal=causal, window=window, stream=stream())
        for b in range(0, batch, 3):
            close(out[b], *exact(q[b], k[b], v[b], 0, tokens // 2 + 100, causal, window), "sequence %d" % b)


class Sequences:
    """Four sequences of n tokens in a cache, the last `new` of each as the batch."""

    def __init__(self, typ, heads, kv, dim, n, new, k, v):
        self.cache = fa.SequenceCache(STORAGE[typ], 1, heads, kv, dim, 16, 4 * -(-n // 16), 4)
        self.at = torch.arange(4 * n, device="cuda").reshape(4, n)
        for rows, count in ((self.at[:, :n - new].flatten(), n - new), (self.at[:, n - new:].flatten(), new)):
            self.cache.extend([0, 1, 2, 3], [count] * 4, stream=stream())
            self.cache.write(0, k[rows], v[rows], stream=stream())


@pytest.mark.gpu
@pytest.mark.parametrize("typ", ["f16", "f32"])
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("new", [1, 70])
def test_cache_with_infinite_keys(typ, dim, new):
    heads, kv, n = 32, 4, 200
    q, k, v = values(dim, typ, (4 * new, heads, dim), (4 * n, kv, dim), (4 * n, kv, dim))
    k = infinite_keys(k, q, [s * n + j for s in range(4) for j in (3, 100, 101, 129)])
    c = Sequences(typ, heads, kv, dim, n, new, k, v)
    out = torch.empty_like(q)
    c.cache.attend(0, q, out, stream=stream())
    for s in range(4):
        mine = slice(s * new, (s + 1) * new)
        close(out[mine], *exact(q[mine], k[c.at[s]], v[c.at[s]], n - new, n // 2 + 100), "sequence %d" % s)


def infinite_values(v, bad):
    """Infinities in the tokens of `bad`, {token: {dim: value}}, of the first key head."""
    v = v.clone()
    for j, x in bad.items():
        for d, y in x.items():
            v[..., j, 0, d] = y
    return v


def check_infinite(got, want, tol, seen, v, what):
    """Where a row sees infinities of one sign in a dim that is the result, with both or a NaN it is NaN; elsewhere it is as if there were none.
    got, want, tol [m, heads, dim]; seen [m, n]; v [n, heads, dim]."""
    count = lambda x: torch.einsum("mn,nhd->mhd", seen.double(), x.double()) > 0   # noqa: E731
    up, down, nan = count(v == math.inf), count(v == -math.inf), count(torch.isnan(v))
    got = got.detach().cpu().double()
    odd = nan | (up & down)
    assert torch.isnan(got[odd]).all(), what
    assert (got[up & ~odd] == math.inf).all() and (got[down & ~odd] == -math.inf).all(), what
    rest = ~(up | down | nan)
    assert ((got - want).abs() <= tol)[rest].all(), what


BAD = {3: {0: math.inf, 5: -math.inf, 7: math.nan}, 20: {0: math.inf, 5: math.inf, 6: -math.inf}, 61: {1: -math.inf, 6: math.inf, 0: math.inf}}


@pytest.mark.gpu
@pytest.mark.parametrize("typ", ["f16", "f32"])
@pytest.mark.parametrize("dim", [8, 40, 64, 80, 128, 200])
@pytest.mark.parametrize("batch,tokens,heads", SIZES)
def test_prompt_with_infinite_values(typ, dim, batch, tokens, heads):
    q, k, v = values(dim, typ, (batch, tokens, heads, dim), (batch, tokens, 2, dim), (batch, tokens, 2, dim))
    bad = infinite_values(v, BAD)
    i, j = torch.arange(tokens)[:, None], torch.arange(tokens)[None, :]
    for causal, window in ((True, 0), (False, 0), (False, 30)):
        out = torch.empty_like(q)
        fa.attention(q, k, bad, out, causal=causal, window=window, stream=stream())
        for b in range(0, batch, 3):
            want, tol = exact(q[b], k[b], v[b], 0, tokens // 2 + 100, causal, window)
            check_infinite(out[b], want, tol, visible(i, j, tokens, causal, window, 0).expand(tokens, tokens), bad[b].cpu().repeat_interleave(heads // 2, 1), "sequence %d" % b)


@pytest.mark.gpu
@pytest.mark.parametrize("typ", ["f16", "f32"])
@pytest.mark.parametrize("dim", [8, 40, 64, 80, 128, 200])
@pytest.mark.parametrize("new,n", [(1, 200), (1, 2500), (70, 200), (130, 300)])
def test_cache_with_infinite_values(typ, dim, new, n):
    heads, kv = 32, 4
    q, k, v = values(dim, typ, (4 * new, heads, dim), (4 * n, kv, dim), (4 * n, kv, dim))
    bad = infinite_values(v, {s * n + j: x for s in range(4) for j, x in BAD.items()})
    c = Sequences(typ, heads, kv, dim, n, new, k, bad)
    out = torch.empty_like(q)
    c.cache.attend(0, q, out, stream=stream())
    i, j = torch.arange(n - new, n)[:, None], torch.arange(n)[None, :]
    for s in range(4):
        mine = slice(s * new, (s + 1) * new)
        want, tol = exact(q[mine], k[c.at[s]], v[c.at[s]], n - new, n // 2 + 100)
        check_infinite(out[mine], want, tol, visible(i, j, n, True, 0, 0), bad[c.at[s]].cpu().repeat_interleave(heads // kv, 1), "sequence %d" % s)


@pytest.mark.gpu
@pytest.mark.parametrize("typ", ["f16", "f32"])
def test_branches_with_infinite_values(typ):
    """... over the pages that branches have in common, and behind them."""
    heads, kv, dim, n, branches = 8, 2, 64, 1300, 5
    q, k, v, nk, nv = values(2, typ, (branches, heads, dim), (n, kv, dim), (n, kv, dim), (branches, kv, dim), (branches, kv, dim))
    bad, nbad = infinite_values(v, {700: {0: math.inf, 5: -math.inf, 7: math.inf}}), infinite_values(nv, {2: {7: -math.inf, 9: math.inf}})
    c = fa.SequenceCache(STORAGE[typ], 1, heads, kv, dim, 16, 100, branches)
    c.extend([0], [n], stream=stream())
    c.write(0, k, bad, stream=stream())
    c.fork(0, list(range(1, branches)), stream=stream())
    c.extend(list(range(branches)), [1] * branches, stream=stream())
    c.write(0, nk, nbad, stream=stream())
    out = torch.empty_like(q)
    c.attend(0, q, out, stream=stream())
    for s in range(branches):
        ks, vs, bs = torch.cat([k, nk[s:s + 1]]), torch.cat([v, nv[s:s + 1]]), torch.cat([bad, nbad[s:s + 1]])
        check_infinite(out[s:s + 1], *exact(q[s:s + 1], ks, vs, n, 200), torch.ones(1, n + 1), bs.cpu().repeat_interleave(heads // kv, 1), "branch %d" % s)


@pytest.mark.gpu
@pytest.mark.parametrize("typ", ["f16", "f32"])
@pytest.mark.parametrize("heads,kv", [(2, 2), (32, 4)])
def test_infinite_values_of_little_weight(typ, heads, kv):
    """Weights of exp(-320), which are zero in 32 bits, of all of a cache's keys but the last ones, which lie in other parts of the row; and of a prompt's."""
    dim, n = 64, 2500
    q, k, v = (torch.ones(m, h, dim, dtype=TYPES[typ], device="cuda") for m, h in ((4, heads), (4 * n, kv), (4 * n, kv)))
    at = torch.arange(4 * n, device="cuda").reshape(4, n)
    k[at[:, :n - 300].flatten()] = -40.0
    v[at[:, 700], :, 1], v[at[:, 1900], :, 2], v[at[:, 30], :, 3], v[at[:, n - 5], :, 3] = math.inf, -math.inf, math.inf, -math.inf
    c = Sequences(typ, heads, kv, dim, n, 1, k, v)
    out = torch.empty_like(q)
    c.cache.attend(0, q, out, stream=stream())
    many = torch.ones(1, n, heads, dim, dtype=q.dtype, device="cuda")
    whole = torch.empty_like(many)
    fa.attention(many, k[:n][None], v[:n][None], whole, causal=False, stream=stream())
    for got in (out, whole[0]):
        assert (got[..., 1] == math.inf).all() and (got[..., 2] == -math.inf).all() and torch.isnan(got[..., 3]).all()
        rest = torch.cat([got[..., :1], got[..., 4:]], -1)
        assert ((rest - 1).abs() <= (2.0 ** -11 if typ == "f16" else 1e-4)).all()   # (sums of ones: the weights' own sum, rounded 300 / 128 + 100 times)
