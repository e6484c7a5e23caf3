"""Sizes at the ends of what the calls on sequences take.  No GPU is asked before an argument is."""
import ctypes

import pytest

import fyusenet_amd as fa
from fyusenet_amd import capi


@pytest.mark.parametrize("pages,page_tokens", [(2048, 1024), (2049, 1024), (1 << 18, 8), ((1 << 18) + 1, 8), (1 << 20, 1024)])
def test_cache_refuses_sizes_beyond_64_bits(pages, page_tokens):
    """Pages of 2^53 or 2^46 bytes, so many of them that the product is 2^64 (zero in 64 bits) or a little more."""
    d = capi.CacheDesc(ctypes.sizeof(capi.CacheDesc), capi.STORAGE_F32, 65536, 65536, 65536, 256, page_tokens, pages, 1, 8)
    h = ctypes.c_void_p()
    with pytest.raises(fa.FynException) as e:
        capi.check(capi.lib().fyn_cache_create(0, ctypes.byref(d), ctypes.byref(h)))
    assert e.value.code == capi.ERR_INVALID and "addressed" in str(e.value) and not h.value


def test_attention_refuses_more_tokens_than_can_be_counted():
    """Positions are 32 bits, with room for the end of the last tile: beyond that nothing is computed, and not silently."""
    for batch, tokens in ((1, 2 ** 31 - 1), (1, 2 ** 31 - 100), (3, 715827882)):
        d = capi.AttentionDesc()
        d.struct_size, d.storage, d.batch, d.tokens, d.heads, d.kv_heads, d.head_dim = ctypes.sizeof(d), capi.STORAGE_F16, batch, tokens, 1, 1, 8
        with pytest.raises(fa.FynException) as e:
            capi.check(capi.lib().fyn_attention(ctypes.byref(d), None))
        assert e.value.code == capi.ERR_INVALID and "%d sequences of %d tokens" % (batch, tokens) in str(e.value)


@pytest.mark.gpu
@pytest.mark.parametrize("batch,tokens,heads,kv_heads", [(300000, 1, 64, 8), (530000, 2, 32, 32)])
def test_more_sequences_than_a_launch_takes(batch, tokens, heads, kv_heads):
    """Nineteen and seventeen million workgroups; a launch has fewer than 2^32 threads."""
    torch = pytest.importorskip("torch")
    gen = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn(batch, tokens, h, 8, generator=gen, device="cuda", dtype=torch.float16) for h in (heads, kv_heads, kv_heads))
    out = torch.full_like(q, 9.0)
    fa.attention(q, k, v, out, causal=True, stream=torch.cuda.current_stream().cuda_stream)
    # a sequence's first token sees itself alone
    assert torch.equal(out[:, 0], v[:, 0].repeat_interleave(heads // kv_heads, 1))
    if tokens > 1:
        s = [(q[:, 1].float() * k[:, j].float()).sum(-1) / 8 ** 0.5 for j in (0, 1)]
        w = torch.sigmoid(s[1] - s[0])[..., None]
        want = (1 - w) * v[:, 0].float() + w * v[:, 1].float()
        # (the weights to 2^-17 or so, and the result's rounding)
        assert ((out[:, 1].float() - want).abs() <= 2.0 ** -14 + 2.0 ** -11 * want.abs()).all()


@pytest.mark.gpu
def test_more_sequences_of_a_cache_than_a_launch_takes():
    torch = pytest.importorskip("torch")
    n, heads = 70000, 256
    s = torch.cuda.current_stream().cuda_stream
    cache = fa.SequenceCache(fa.STORAGE_F16, 1, heads, heads, 8, 8, n, n, 8)
    gen = torch.Generator(device="cuda").manual_seed(2)
    q, k, v = (torch.randn(n, heads, 8, generator=gen, device="cuda", dtype=torch.float16) for _ in range(3))
    out = torch.full_like(q, 9.0)
    who = list(range(n))
    cache.extend(who, [1] * n, stream=s)
    cache.write(0, k, v, stream=s)
    cache.attend(0, q, out, stream=s)
    assert torch.equal(out, v)
    cache.extend(who[::-1], [1] * n, stream=s)      # (each has itself and one before: the same value twice)
    cache.write(0, q.flip(0), v.flip(0), stream=s)
    cache.attend(0, q.flip(0), out, stream=s)
    assert ((out.float() - v.flip(0).float()).abs() <= 2.0 ** -11 * v.flip(0).float().abs() + 2.0 ** -24).all()
    cache.close()


class _Unopened(fa.SequenceCache):
    """The Python side of a cache whose handle is null: what it refuses by itself."""

    def __init__(self):
        self._h, self.kv_heads, self.head_dim, self.heads, self._type = ctypes.c_void_p(), 1, 8, 1, "float16"


@pytest.mark.parametrize("far", [2 ** 32, 2 ** 32 + 1, 2 ** 31, -2 ** 31 - 1, 2 ** 64])
def test_python_refuses_numbers_beyond_32_bits(far):
    """... instead of taking their last 32 bits: sequence 2^32 is not sequence 0."""
    c, x = _Unopened(), fa.DeviceArray(1 << 20, "float16", (3, 1, 8))
    b = fa.AttentionLayerBuilder(1, 1, 8, "mix").window(far)
    for call in (lambda: c.extend([far], [1]), lambda: c.extend([0], [far]), lambda: c.fork(far, [1]), lambda: c.fork(0, [far]), lambda: c.fork(0, [1], far),
                 lambda: c.copy([0], [far]), lambda: c.extend(list(range(20)) + [far], [1] * 21), lambda: c.free([3] * 12 + [far]), lambda: c.truncate([0], [far]), lambda: c.free([far]), lambda: c.lengths([far]), lambda: c.write(far, x, x),
                 lambda: c.attend(far, x, x), lambda: c.read([far], 0, x, x), lambda: c.read([0], far, x, x), b.attention,
                 lambda: fa.SequenceCache(fa.STORAGE_F16, 1, 1, 1, 8, 8, far, 1), lambda: fa.SequenceCache(fa.STORAGE_F16, 1, 1, 1, 8, 8, 1, 1, far)):
        with pytest.raises(fa.FynException) as e:
            call()
        assert e.value.code == capi.ERR_INVALID and "null" not in str(e.value) and "cache:" not in str(e.value)


#   shape [batch, tokens, heads, 8], strides
OVERLAPPING = [((2, 3, 4, 8), (0, 32, 8, 1)), ((2, 3, 4, 8), (96, 0, 8, 1)), ((2, 3, 4, 8), (96, 32, 0, 1)), ((2, 3, 4, 8), (96, 24, 8, 1)), ((2, 3, 4, 8), (88, 32, 8, 1)),
               ((1, 3, 1, 8), (0, 0, 0, 1))]
APART = [((2, 3, 4, 8), (96, 32, 8, 1)), ((2, 3, 4, 8), (8, 64, 16, 1)), ((2, 3, 4, 8), (96, 8, 24, 1)), ((1, 3, 1, 8), (0, 16, 0, 1)), ((1, 1, 1, 8), (0, 0, 0, 1))]


@pytest.mark.parametrize("shape,strides", OVERLAPPING + APART)
def test_results_that_overlap_are_refused(shape, strides):
    """(The addresses here are nobody's: what is refused for its rows is refused in front of that.)"""
    q = fa.DeviceArray(1 << 20, "float16", shape)
    with pytest.raises(fa.FynException) as e:
        fa.attention(q, q, q, fa.DeviceArray(1 << 24, "float16", shape, strides))
    assert e.value.code == capi.ERR_INVALID and ("overlap" in str(e.value)) == ((shape, strides) in OVERLAPPING)


@pytest.mark.gpu
def test_results_of_a_cache_that_overlap_are_refused():
    torch = pytest.importorskip("torch")
    s = torch.cuda.current_stream().cuda_stream
    c = fa.SequenceCache(fa.STORAGE_F16, 1, 4, 2, 8, 8, 4, 2)
    kv, q = torch.ones(3, 2, 8, dtype=torch.float16, device="cuda"), torch.ones(3, 4, 8, dtype=torch.float16, device="cuda")
    c.extend([0], [3], stream=s)
    c.write(0, kv[:1].expand(3, 2, 8), kv[:, :1].expand(3, 2, 8), stream=s)     # (what is read may be the same for all)
    out, back = torch.zeros_like(q), torch.zeros_like(kv)
    for call in (lambda: c.attend(0, q, out[:1].expand(3, 4, 8)), lambda: c.attend(0, q, out[:, :1].expand(3, 4, 8)),
                 lambda: c.read([0], 0, back[:1].expand(3, 2, 8), torch.zeros_like(kv)), lambda: c.read([0], 0, torch.zeros_like(kv), back[:, :1].expand(3, 2, 8))):
        with pytest.raises(fa.FynException) as e:
            call()
        assert "overlap" in str(e.value)
    c.attend(0, q[:1].expand(3, 4, 8), out, stream=s)
    c.read([0], 0, back, torch.zeros_like(kv), stream=s)
    assert (out == 1).all() and (back == 1).all()
