"""Keys that are infinite and seen: a score of minus infinity is a weight of zero, whatever the size of a head.  Tolerances: tests/test_gpu_sequences_precision.py."""
import math

import pytest

import fyusenet_amd as fa
from tests.test_gpu_sequences import STORAGE, close, stream, values
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
