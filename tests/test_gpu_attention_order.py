"""The order between a cache's calls and what else works on it."""
import numpy as np
import pytest

import fyusenet_amd as fa
from fyusenet_amd import capi
from tests.test_gpu_sequences import close
from tests.test_gpu_sequences_precision import exact
from tests.util import make_single_layer_net

torch = pytest.importorskip("torch")


def behind_something_long(side):
    """Work of some milliseconds on a stream: what is queued behind it is late."""
    with torch.cuda.stream(side):
        a = torch.ones(8192, 8192, device="cuda")
        for _ in range(6):
            a = torch.mm(a, a).clamp_(max=1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("storage", [fa.STORAGE_F32, fa.STORAGE_F16], ids=["f32", "f16"])
def test_timing_a_layer_waits_for_the_cache(storage):
    """A layer that is bound to a cache is timed right behind changes of the cache on another stream: its new tokens go where these say."""
    heads, kv, dim, n = 4, 2, 32, 3
    typ = torch.float16 if storage == fa.STORAGE_F16 else torch.float32
    cache = fa.SequenceCache(storage, 1, heads, kv, dim, 8, 60, 6)
    net = make_single_layer_net(fa.AttentionLayerBuilder(heads, kv, dim, "mix").number(1).deep().size(n, 1).causal(), storage)
    net.layers[1].bindCache(cache)
    rng = np.random.default_rng(2)
    ins = [rng.standard_normal((c * dim, 1, n)).astype(np.float32) for c in (heads, kv, kv)]
    for port, x in enumerate(ins):
        net.layers[1].setInput(x, port)
    new = [torch.from_numpy(x[:, 0].T.reshape(n, kv, dim).copy()).to(typ).cuda() for x in ins[1:]]
    side, gen = torch.cuda.Stream(), torch.Generator().manual_seed(4)
    old = [[torch.randn(20 + 5 * s, kv, dim, generator=gen).to(typ).cuda() for s in range(3)] for _ in range(2)]
    torch.cuda.synchronize()
    cache.extend([0, 1, 2], [20, 25, 30], stream=side.cuda_stream)
    cache.write(0, torch.cat(old[0]), torch.cat(old[1]), stream=side.cuda_stream)
    have = {s: [old[0][s], old[1][s]] for s in range(3)}
    for who, counts in (([0, 1, 2], [1, 1, 1]), ([2], [3]), ([1, 0], [1, 2])):
        torch.cuda.synchronize()
        behind_something_long(side)
        cache.free([2], stream=side.cuda_stream)                  # (its pages go to others)
        cache.extend(who, counts, stream=side.cuda_stream)
        have[2] = [x[:0] for x in have[2]]
        assert net.layers[1].timeKernel(3) > 0
        at = 0
        for s, m in zip(who, counts):
            have[s] = [torch.cat([x, y[at:at + m]]) for x, y in zip(have[s], new)]
            at += m
        rows = sum(cache.lengths([0, 1, 2]))
        got = [torch.empty(rows, kv, dim, dtype=typ, device="cuda") for _ in range(2)]
        cache.read([0, 1, 2], 0, *got, stream=side.cuda_stream)
        torch.cuda.synchronize()
        for x, y in zip(got, range(2)):
            assert torch.equal(x, torch.cat([have[s][y] for s in range(3)]))
    cache.extend([1], [1], stream=side.cuda_stream)               # a batch of another size: refused, as a pass is
    with pytest.raises(fa.FynException) as e:
        net.layers[1].timeKernel(3)
    assert e.value.code == capi.ERR_INVALID
    net.layers[1].bindCache(None)
    assert net.layers[1].timeKernel(3) > 0
    net.cleanup()


@pytest.mark.gpu
def test_replays_in_order():
    """A captured step on a stream of its own, put in order by fyn_cache_order in front of each replay, between calls on others; under capture
    there is no order to be had, and that is said."""
    heads, kv, dim, n = 4, 2, 64, 3
    cache = fa.SequenceCache(fa.STORAGE_F16, 1, heads, kv, dim, 16, 400, n)
    gen = torch.Generator().manual_seed(3)
    k, v, q = (torch.randn(n, h, dim, generator=gen).half().cuda() for h in (kv, kv, heads))
    out, side, mine = torch.zeros_like(q), torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    old = [torch.randn(n * 100, kv, dim, generator=gen).half().cuda() for _ in range(2)]
    torch.cuda.synchronize()
    cache.extend([0, 1, 2], [100] * n, stream=side.cuda_stream)
    cache.write(0, *old, stream=side.cuda_stream)
    have = [[x[s * 100:(s + 1) * 100] for x in old] for s in range(n)]
    cache.extend([0, 1, 2], [1] * n, stream=side.cuda_stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=mine):
        cache.write(0, k, v, stream=mine.cuda_stream)
        cache.attend(0, q, out, stream=mine.cuda_stream)
        with pytest.raises(fa.FynException) as e:
            cache.order(mine.cuda_stream)
        assert e.value.code == capi.ERR_STATE
    for turn in range(4):
        if turn:
            behind_something_long(side)
            cache.extend([0, 1, 2], [1] * n, stream=side.cuda_stream)
        cache.order(mine.cuda_stream)
        with torch.cuda.stream(mine):
            graph.replay()
        rows = sum(cache.lengths([0, 1, 2]))
        have = [[torch.cat([x, y[s:s + 1]]) for x, y in zip(have[s], (k, v))] for s in range(n)]
        got = [torch.empty(rows, kv, dim, dtype=torch.float16, device="cuda") for _ in range(2)]
        torch.cuda.current_stream().synchronize()
        cache.read([0, 1, 2], 0, *got, stream=side.cuda_stream)    # (behind the replay)
        cache.order(torch.cuda.current_stream().cuda_stream)
        for i, x in enumerate(got):
            assert torch.equal(x, torch.cat([have[s][i] for s in range(n)]))
        for s in range(n):
            close(out[s:s + 1], *exact(q[s:s + 1], *have[s], have[s][0].shape[0] - 1, 100))
        torch.cuda.synchronize()
