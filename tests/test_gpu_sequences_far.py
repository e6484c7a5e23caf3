"""Attention and the cache at distances beyond 32 bits, and captured attention of prompts.  Tolerances: tests/test_gpu_sequences_precision.py."""
import pytest

import fyusenet_amd as fa
from tests.test_gpu_sequences import STORAGE, TYPES, close, stream, values
from tests.test_gpu_sequences_precision import exact

torch = pytest.importorskip("torch")


@pytest.mark.gpu
@pytest.mark.parametrize("typ,pitch", [("f16", 1 << 23), ("f16", (1 << 23) + 8), ("f32", 1 << 22), ("f32", (1 << 22) + 4)])
@pytest.mark.parametrize("heads", [2, 48])
def test_tokens_far_apart(typ, pitch, heads):
    """Keys and values 16 MB apart, 5 GB in all: the largest distance that goes through tiles, and one more."""
    tokens, dim = 330, 64
    both = torch.empty(tokens * pitch, dtype=TYPES[typ], device="cuda")
    k, v = (both.as_strided((1, tokens, 2, dim), (0, pitch, dim, 1), at) for at in (0, 2 * dim))
    q, k0, v0 = values(6, typ, (1, tokens, heads, dim), (1, tokens, 2, dim), (1, tokens, 2, dim))
    k.copy_(k0)
    v.copy_(v0)
    for causal, window in ((True, 0), (False, 100)):
        out = torch.empty_like(q)
        fa.attention(q, k, v, out, causal=causal, window=window, stream=stream())
        close(out[0], *exact(q[0], k0[0], v0[0], 0, tokens // 2 + 100, causal, window))


@pytest.mark.gpu
@pytest.mark.parametrize("typ", ["f16", "f32"])
def test_pages_far_into_a_cache(typ):
    """Sequences whose pages begin behind 5 GB of another's: written, attended to, read, branched, copied and moved."""
    heads, kv, dim, page, layers = 32, 8, 128, 16, 2
    each = layers * 2 * kv * dim * (2 if typ == "f16" else 4)
    far = 5 * 2 ** 30 // each // page * page
    cache = fa.SequenceCache(STORAGE[typ], layers, heads, kv, dim, page, far // page + 200, 6)
    cache.extend([0], [far], stream=stream())
    want = {}
    for s, before, new in ((1, 400, 1), (2, 90, 70)):
        k, v, q = values(s, typ, (layers, before + new, kv, dim), (layers, before + new, kv, dim), (layers, new, heads, dim))
        want[s] = (k, v)
        for at, count in ((0, before), (before, new)):
            cache.extend([s], [count], stream=stream())
            for i in range(layers):
                cache.write(i, k[i, at:at + count], v[i, at:at + count], stream=stream())
        for i in range(layers):
            out = torch.empty_like(q[i])
            cache.attend(i, q[i], out, stream=stream())
            close(out, *exact(q[i], k[i], v[i], before, 200), "sequence %d" % s)
    cache.fork(1, [3], 395, stream=stream())
    cache.copy([2], [4], stream=stream())
    want[3], want[4] = (want[1][0][:, :395], want[1][1][:, :395]), want[2]
    k, v = values(9, typ, (layers, 1, kv, dim), (layers, 1, kv, dim))
    cache.extend([3], [1], stream=stream())          # (its last page is copied)
    for i in range(layers):
        cache.write(i, k[i], v[i], stream=stream())
    want[3] = [torch.cat([x, y], 1) for x, y in zip(want[3], (k, v))]

    def check():
        who = [4, 1, 3, 2]
        rows = sum(cache.lengths(who))
        for i in range(layers):
            got = [torch.empty(rows, kv, dim, dtype=TYPES[typ], device="cuda") for _ in range(2)]
            cache.read(who, i, *got, stream=stream())
            for x, y in zip(got, range(2)):
                assert torch.equal(x, torch.cat([want[s][y][i] for s in who]))

    check()
    cache.free([0], stream=stream())
    cache.compact(stream=stream())
    check()
    cache.close()


@pytest.mark.gpu
@pytest.mark.parametrize("typ", ["f16", "f32"])
@pytest.mark.parametrize("batch,tokens,heads,dim", [(2, 60, 4, 40), (4, 130, 32, 64), (6, 160, 48, 64)])   # (sixteen columns, 64 and 128 queries a workgroup)
def test_captured_prompts(typ, batch, tokens, heads, dim):
    """Captured once and replayed with other tensors' contents and other lengths, with eager calls in between."""
    q, k, v = values(1, typ, (batch, tokens, heads, dim), (batch, tokens, 2, dim), (batch, tokens, 2, dim))
    lengths = torch.full((batch,), tokens, dtype=torch.int32, device="cuda")
    out = torch.empty_like(q)

    def call(result):
        fa.attention(q, k, v, result, lengths=lengths, window=50, sinks=2, stream=stream())

    call(out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out)
    for turn in range(4):
        for a, b in zip((q, k, v), values(10 + turn, typ, q.shape, k.shape, v.shape)):
            a.copy_(b)
        n = [max(0, tokens - 37 * turn * b) for b in range(batch)]
        lengths.copy_(torch.tensor(n, dtype=torch.int32))
        out.fill_(5.0)
        graph.replay()
        eager = torch.empty_like(out)
        call(eager)
        assert torch.equal(out, eager)
        for b in range(batch):
            close(out[b, :n[b]], *exact(q[b, :n[b]], k[b, :n[b]], v[b, :n[b]], 0, tokens // 2 + 100, True, 50, 2)) if n[b] else None
            assert (out[b, n[b]:] == 0).all()
        torch.cuda.synchronize()
