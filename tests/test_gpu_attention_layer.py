"""The attention layer in networks: between the positions of a map, between those of its rows, and over a cache; against the
formula in 64 bits on the layer's own inputs (tolerances: tests/test_gpu_sequences.py)."""
import ctypes

import numpy as np
import pytest

import fyusenet_amd as fa
from fyusenet_amd import capi
from tests.test_gpu_sequences import close, reference
from tests.util import conv_block, make_single_layer_net

torch = pytest.importorskip("torch")

STORAGES = [pytest.param(fa.STORAGE_F32, id="f32"), pytest.param(fa.STORAGE_F16, id="f16")]


def builder(heads=4, kv=2, dim=32, width=9, height=7, number=1):
    return fa.AttentionLayerBuilder(heads, kv, dim, "mix").number(number).deep().size(width, height)


def tokens(chw, heads, storage):
    """[channels, height, width] as a layer's tensor has it -> [height, width, heads, dim] of the storage type."""
    c, h, w = chw.shape
    x = torch.from_numpy(np.ascontiguousarray(chw.transpose(1, 2, 0))).reshape(h, w, heads, c // heads)
    return x.half() if storage == fa.STORAGE_F16 else x


@pytest.mark.gpu
@pytest.mark.parametrize("storage", STORAGES)
@pytest.mark.parametrize("rows,causal,window,sinks,padding", [(False, False, 0, 0, 0), (False, True, 11, 3, 0), (True, False, 0, 0, 0), (True, True, 4, 1, 1), (True, False, 3, 0, 2)])
def test_attention_layer(storage, rows, causal, window, sinks, padding):
    heads, kv, dim, w, h = 4, 2, 40, 19, 7
    b = builder(heads, kv, dim, w, h).window(window, sinks).scoreScale(0.3).inputPadding(padding).outputPadding(padding)
    if causal:
        b.causal()
    if rows:
        b.rowsAreSequences()
    net = make_single_layer_net(b, storage)
    lyr = net.layers[1]
    rng = np.random.default_rng(3)
    typ = np.float16 if storage == fa.STORAGE_F16 else np.float32
    ins = [rng.standard_normal((n * dim, h, w)).astype(typ).astype(np.float32) for n in (heads, kv, kv)]
    for port, x in enumerate(ins):
        lyr.setInput(x, port)
    for graph in (False, True):
        net.useGraph(graph)
        for _ in range(2):
            net.forward()
            net.finish()
        out = lyr.copyResult(includePadding=True)
        inner = out[:, padding:padding + h, padding:padding + w]
        assert np.count_nonzero(out) == np.count_nonzero(inner)   # the halo stays zero
        q, k, v = (tokens(x, n, storage) for x, n in zip(ins, (heads, kv, kv)))
        got = tokens(inner, heads, storage)
        if rows:
            for y in range(h):
                close(got[y], *reference(q[y], k[y], v[y], 0, causal, window, sinks, 0.3))
        else:
            close(got.reshape(h * w, heads, dim), *reference(*(x.reshape(h * w, -1, dim) for x in (q, k, v)), 0, causal, window, sinks, 0.3))
    net.cleanup()


class Block(fa.NeuralNetwork):
    """1x1 convolutions to queries, keys and values, causal attention, a 1x1 convolution on its result that adds the input, and the channel
    that is largest at each position: what a network that goes on with a sequence does for a token."""
    HEADS, KV, DIM, CHANNELS = 4, 2, 32, 48

    def __init__(self, storage, width, height):
        super().__init__(storage)
        self.w, self.h = width, height

    def buildLayers(self, factory):
        c, a, k = self.CHANNELS, self.HEADS * self.DIM, self.KV * self.DIM

        def pointwise(no, cin, cout, name):
            return fa.ConvLayerBuilder(1, name).number(no).shape(cout, self.h, self.w, cin).deep()
        pointwise(1, c, c, "in").push(factory)
        for no, n in ((2, a), (3, k), (4, k)):
            pointwise(no, c, n, "p%d" % no).push(factory)
        builder(self.HEADS, self.KV, self.DIM, self.w, self.h, 5).causal().window(40, 2).push(factory)
        pointwise(6, a, c, "back").residual().push(factory)
        fa.ArgMaxLayerBuilder("pick").number(7).shape(c, self.h, self.w, c).deep().push(factory)

    def connectLayers(self, layers, bm):
        for src, dst, port in ((1, 2, 0), (1, 3, 0), (1, 4, 0), (2, 5, 0), (3, 5, 1), (4, 5, 2), (5, 6, 0), (1, 6, 1), (6, 7, 0)):
            bm.connectLayers(layers[src], layers[dst], port)

    def initializeWeights(self, layers):
        c, a, k = self.CHANNELS, self.HEADS * self.DIM, self.KV * self.DIM
        for no, cin, cout in ((1, c, c), (2, c, a), (3, c, k), (4, c, k), (6, a, c)):
            layers[no].loadWeightsAndBiases(conv_block(10 * no, cout, 1, cin), 0)


@pytest.mark.gpu
@pytest.mark.parametrize("storage", STORAGES)
@pytest.mark.parametrize("graph", [False, True], ids=["eager", "graph"])
def test_network_over_a_cache(storage, graph):
    """A prompt of each of three sequences through one network, then single tokens of all of them through another that is bound to the
    same cache; what attention made of them, and the largest channel, against the whole sequences in one pass."""
    heads, kv, dim = Block.HEADS, Block.KV, Block.DIM
    prompt, steps, n = 50, 6, 3
    rng = np.random.default_rng(5)
    x = rng.standard_normal((n, Block.CHANNELS, 1, prompt + steps)).astype(np.float32)
    cache = fa.SequenceCache(storage, 2, heads, kv, dim, 16, 40, n + 1)
    whole, first, step = Block(storage, prompt + steps, 1), Block(storage, prompt, 1), Block(storage, n, 1)
    for net in (whole, first, step):
        net.setup(reuseBuffers=False)
        net.useGraph(graph)
    for net in (first, step):
        net.layers[5].bindCache(cache, 1)
    cache.close()   # (the networks keep it)
    cache = None
    with pytest.raises(fa.FynException):   # nothing has been asked of the cache: no new tokens
        first.forward()
    net_cache = fa.SequenceCache(storage, 1, heads, kv, dim, 16, 40, n + 1)
    for net in (first, step):
        net.layers[5].bindCache(net_cache, 0)
    typ = torch.float16 if storage == fa.STORAGE_F16 else torch.float32
    made = [[] for _ in range(n)]

    def look(net, who, rows):
        """Result of attention at the new tokens against queries and what the cache has."""
        net.finish()
        q = tokens(net.layers[2].copyResult(), heads, storage)[0]
        out = tokens(net.layers[5].copyResult(), heads, storage)[0]
        at = 0
        for s, m in zip(who, rows):
            have = net_cache.lengths([s])[0]
            k, v = (torch.empty(have, kv, dim, dtype=typ, device="cuda") for _ in range(2))
            net_cache.read([s], 0, k, v, stream=torch.cuda.current_stream().cuda_stream)
            close(out[at:at + m], *reference(q[at:at + m], k, v, have - m, True, 40, 2))
            made[s].append(net.layers[6].copyResult()[:, 0, at:at + m])
            at += m

    for s in range(n):
        net_cache.extend([s], [prompt])
        first.layers[1].setInput(x[s, :, :, :prompt])
        first.forward()
        look(first, [s], [prompt])
    for i in range(steps):
        net_cache.extend(list(range(n)), [1] * n)
        step.layers[1].setInput(x[:, :, 0, prompt + i].T.reshape(Block.CHANNELS, 1, n))
        step.forward()
        look(step, list(range(n)), [1] * n)
    for s in range(n):
        whole.layers[1].setInput(x[s])
        whole.forward()
        whole.finish()
        want = whole.layers[6].copyResult()[:, 0]
        got = np.concatenate(made[s], 1)
        # (the convolutions' kernels differ with the maps' sizes: their own accuracy, as tests/test_gpu_conv.py has it)
        assert np.linalg.norm(got - want) <= (2e-3 if storage == fa.STORAGE_F16 else 1e-4) * np.linalg.norm(want)
        idx, _ = whole.getArgMax(7)
        sure = np.sort(want, 0)[-1] - np.sort(want, 0)[-2] > (0.05 if storage == fa.STORAGE_F16 else 1e-3)
        assert (got.argmax(0)[sure] == idx[0][sure]).all()
    # a branch through the network, and the layer as it was described
    net_cache.fork(1, [3])
    net_cache.extend([3, 0, 2], [1, 1, 1])
    step.forward()
    look_lengths = net_cache.lengths([0, 1, 2, 3])
    assert look_lengths == [prompt + steps + 1, prompt + steps, prompt + steps + 1, prompt + steps + 1]
    net_cache.extend([0], [1])
    with pytest.raises(fa.FynException) as e:   # a pass of three positions over a batch of one token
        step.forward()
    assert e.value.code == capi.ERR_INVALID
    step.layers[5].bindCache(None)
    step.forward()
    step.finish()
    q, k, v = (tokens(step.layers[i].copyResult(), m, storage)[0] for i, m in ((2, heads), (3, kv), (4, kv)))
    close(tokens(step.layers[5].copyResult(), heads, storage)[0], *reference(q, k, v, 0, True, 40, 2))
    for net in (whole, first, step):
        net.cleanup()


@pytest.mark.gpu
@pytest.mark.parametrize("storage", STORAGES)
def test_captured_pass_follows_the_batch(storage):
    """The same network, captured, over batches of the same number of tokens that are divided differently; bound before it is set up."""
    heads, kv, dim, rows = 4, 2, 32, 6
    cache = fa.SequenceCache(storage, 1, heads, kv, dim, 8, 60, 6)

    class Net(fa.NeuralNetwork):
        def buildLayers(self, factory):
            builder(heads, kv, dim, rows, 1).causal().push(factory)

        def connectLayers(self, layers, bm):
            layers[1].bindCache(cache)

    net = Net(storage)
    net.setup()
    net.useGraph(True)
    typ = np.float16 if storage == fa.STORAGE_F16 else np.float32
    rng = np.random.default_rng(6)
    past = {s: [] for s in range(6)}
    for who, counts in (([0, 1, 2, 3, 4, 5], [1] * 6), ([0, 1, 2, 3, 4, 5], [1] * 6), ([3, 1], [2, 4]), ([2], [6]), ([0, 5, 4], [3, 0, 3]), ([0, 1, 2, 3, 4, 5], [1] * 6)):
        ins = [rng.standard_normal((n * dim, 1, rows)).astype(typ).astype(np.float32) for n in (heads, kv, kv)]
        for port, x in enumerate(ins):
            net.layers[1].setInput(x, port)
        cache.extend(who, counts)
        net.forward()
        net.finish()
        got = tokens(net.layers[1].copyResult(), heads, storage)[0]
        q, k, v = (tokens(x, n, storage)[0] for x, n in zip(ins, (heads, kv, kv)))
        at = 0
        for s, m in zip(who, counts):
            past[s].append((k[at:at + m], v[at:at + m]))
            ks, vs = (torch.cat([x[i] for x in past[s]]) for i in (0, 1))
            close(got[at:at + m], *reference(q[at:at + m], ks, vs, ks.shape[0] - m))
            at += m
    net.cleanup()


@pytest.mark.gpu
def test_attention_layer_in_a_network_with_buffer_reuse():
    """The same block with and without shared buffers, eager and from the captured graph: the same bits."""
    x = np.random.default_rng(8).standard_normal((Block.CHANNELS, 12, 31)).astype(np.float32)
    got = []
    for reuse in (False, True):
        for graph in (False, True):
            net = Block(fa.STORAGE_F16, 31, 12)
            net.setup(reuseBuffers=reuse)
            net.useGraph(graph)
            for _ in range(3):
                net.layers[1].setInput(x)
                net.forward()
                net.finish()
            got.append(net.getArgMax(7)[0])
            net.cleanup()
    assert all((g == got[0]).all() for g in got)


def _refused(net_builder, storage=fa.STORAGE_F16):
    d, a = net_builder.desc(), net_builder.attention()
    h = ctypes.c_void_p()
    capi.check(capi.lib().fyn_net_create(0, storage, ctypes.byref(h)))
    try:
        assert capi.lib().fyn_net_add_layer(h, ctypes.byref(d)) != capi.OK   # (attention layers have a call of their own)
        return capi.lib().fyn_net_add_attention_layer(h, ctypes.byref(d), ctypes.byref(a))
    finally:
        capi.lib().fyn_net_destroy(h)


@pytest.mark.gpu
def test_attention_layer_refuses():
    assert _refused(builder()) == capi.OK
    assert _refused(builder(dim=20)) == capi.ERR_UNSUPPORTED
    assert _refused(builder(heads=4, kv=3)) == capi.ERR_INVALID
    assert _refused(builder().inputPadding(1)) == capi.ERR_UNSUPPORTED
    assert _refused(builder().window(-1)) == capi.ERR_INVALID
    assert _refused(builder().prefixAct(fa.ActType.RELU)) == capi.ERR_UNSUPPORTED
    assert _refused(builder(width=65535, height=65535)) == capi.ERR_INVALID
    assert _refused(builder().scoreScale(float("inf"))) == capi.ERR_INVALID
    b = builder()
    b.headDim_ = 16
    assert _refused(b) == capi.ERR_INVALID
    net = make_single_layer_net(builder(width=3, height=1), fa.STORAGE_F16)
    good = dict(storage=fa.STORAGE_F16, layers=2, heads=4, kv_heads=2, head_dim=32, page_tokens=16, pages=4, sequences=2)
    with pytest.raises(fa.FynException):   # not causal
        net.layers[1].bindCache(fa.SequenceCache(**good))
    net.cleanup()
    net = make_single_layer_net(builder(width=3, height=1).causal(), fa.STORAGE_F16)
    for wrong in ({"storage": fa.STORAGE_F32}, {"heads": 2}, {"kv_heads": 4}, {"head_dim": 40}):
        with pytest.raises(fa.FynException):
            net.layers[1].bindCache(fa.SequenceCache(**dict(good, **wrong)))
    with pytest.raises(fa.FynException):
        net.layers[1].bindCache(fa.SequenceCache(**good), 2)
    net.layers[1].bindCache(fa.SequenceCache(**good), 1)
    net.cleanup()
    padded = make_single_layer_net(builder(width=3, height=1).causal().rowsAreSequences().inputPadding(1), fa.STORAGE_F16)
    with pytest.raises(fa.FynException):
        padded.layers[1].bindCache(fa.SequenceCache(**good))
    padded.cleanup()
    conv = make_single_layer_net(fa.ConvLayerBuilder(1, "c").number(1).shape(8, 4, 4, 8).deep(), fa.STORAGE_F16, weights=np.zeros(72, np.float32))
    with pytest.raises(fa.FynException):
        conv.layers[1].bindCache(fa.SequenceCache(**good))
    conv.cleanup()


@pytest.mark.gpu
def test_custom_layer_calls_attention():
    """A layer of the application that works on tensor views, as custom layers get them."""
    heads, dim, w, h = 2, 16, 21, 3

    class Mix:
        def forward(self, inputs, output, stream, sequence):
            fa.attention(inputs[0], inputs[1], inputs[2], output, causal=True, heads=heads, kv_heads=heads, stream=stream)

    b = fa.CustomLayerBuilder("mix", lambda _: Mix()).number(1).shape(heads * dim, h, w, heads * dim)
    for _ in range(3):
        b.input(heads * dim, 1)
    net = make_single_layer_net(b.outputPadding(2), fa.STORAGE_F32)
    ins = [np.random.default_rng(i).standard_normal((heads * dim, h, w)).astype(np.float32) for i in range(3)]
    for port, x in enumerate(ins):
        net.layers[1].setInput(x, port)
    net.forward()
    net.finish()
    got = tokens(net.layers[1].copyResult(), heads, fa.STORAGE_F32)
    q, k, v = (tokens(x, heads, fa.STORAGE_F32) for x in ins)
    for y in range(h):
        close(got[y], *reference(q[y], k[y], v[y], 0))
    net.cleanup()
