"""The operators on sequences as cases that can be timed and compared: attention over a prompt with a sliding window and
first tokens that stay visible, attention of new tokens over a paged cache, and the management of that cache's pages.

A case names one of four operations:

  prompt    every token of a padded batch attends to its sequence
  decode    one new token for each sequence attends to what the cache holds of it
  fork      one sequence branches: every branch takes a token of its own and attends to the shared past and to that token
  turnover  half of the sequences end, the pages of the others move together, and new sequences start as their copies

run() has two forms: elementary torch operations on tensors of pages, and (own) the calls of this package.
"""
import math
import random

import torch

own = False

TYPES = {"f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # the positions of a 14 x 14 map with one class token in front, both directions, one image: launches count
        {"name": "prompt_197_map_f16", "op": "prompt", "type": "f16", "batch": 1, "tokens": 197, "heads": 12, "kv_heads": 12, "dim": 64,
         "causal": False, "window": 0, "sinks": 0, "ragged": False},
        # prompts of different lengths in one padded batch, shared key heads, a window with four first tokens
        {"name": "prompt_4x2001_window_f16", "op": "prompt", "type": "f16", "batch": 4, "tokens": 2001, "heads": 32, "kv_heads": 8, "dim": 128,
         "causal": True, "window": 512, "sinks": 4, "ragged": True},
        # one long prompt, everything before a token is visible
        {"name": "prompt_16384_causal_f16", "op": "prompt", "type": "f16", "batch": 1, "tokens": 16384, "heads": 16, "kv_heads": 4, "dim": 128,
         "causal": True, "window": 0, "sinks": 0, "ragged": False},
        # 32-bit tensors: a map of 48 x 40 positions with register tokens in front that all positions see
        {"name": "prompt_2x1924_map_f32", "op": "prompt", "type": "f32", "batch": 2, "tokens": 1924, "heads": 8, "kv_heads": 8, "dim": 64,
         "causal": False, "window": 320, "sinks": 4, "ragged": False},
        # one stream at its beginning: the smallest call
        {"name": "decode_1x230_f16", "op": "decode", "type": "f16", "batch": 1, "tokens": 230, "heads": 16, "kv_heads": 4, "dim": 64,
         "window": 0, "sinks": 0, "ragged": False, "page": 16},
        # an ordinary batch of a service, every sequence of another length
        {"name": "decode_24x5000_f16", "op": "decode", "type": "f16", "batch": 24, "tokens": 5000, "heads": 32, "kv_heads": 8, "dim": 128,
         "window": 0, "sinks": 0, "ragged": True, "page": 16},
        # many long sequences: the largest
        {"name": "decode_64x32768_f16", "op": "decode", "type": "f16", "batch": 64, "tokens": 32768, "heads": 32, "kv_heads": 8, "dim": 128,
         "window": 0, "sinks": 0, "ragged": False, "page": 64},
        # endless streams in 32 bits: a window and the first tokens of each
        {"name": "decode_16x20000_window_f32", "op": "decode", "type": "f32", "batch": 16, "tokens": 20000, "heads": 8, "kv_heads": 8, "dim": 96,
         "window": 4096, "sinks": 4, "ragged": True, "page": 32},
        # two answers tried for one short prompt
        {"name": "fork_2x333_f16", "op": "fork", "type": "f16", "branches": 2, "tokens": 333, "heads": 16, "kv_heads": 4, "dim": 64, "page": 16},
        # many answers sampled for one long prompt
        {"name": "fork_32x12005_f16", "op": "fork", "type": "f16", "branches": 32, "tokens": 12005, "heads": 32, "kv_heads": 8, "dim": 128, "page": 32},
        # a small service: two of four sequences end
        {"name": "turnover_4x500_f32", "op": "turnover", "type": "f32", "sequences": 4, "tokens": 500, "kv_heads": 8, "dim": 64, "layers": 2, "page": 16},
        # a large one
        {"name": "turnover_24x9000_f16", "op": "turnover", "type": "f16", "sequences": 24, "tokens": 9000, "kv_heads": 8, "dim": 128, "layers": 4, "page": 32},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "decode", "decode", "fork", "turnover"])
    kv_heads, dim = rng.choice([1, 2, 4, 8]), rng.choice([32, 64, 80, 96, 128])
    c = {"op": op, "type": rng.choice(["f16", "f16", "f32"]), "kv_heads": kv_heads, "dim": dim}
    if op != "turnover":
        c["heads"] = kv_heads * rng.choice([1, 2, 3, 4, 8])
    if op in ("prompt", "decode"):
        c.update(window=0 if rng.random() < 0.5 else _log(rng, 16, 4096), ragged=rng.random() < 0.5)
        c["sinks"] = rng.choice([0, 1, 4, 70]) if c["window"] else 0
    if op == "prompt":
        c["causal"] = rng.random() < 0.6
        c["batch"] = rng.randint(1, 6)
        c["tokens"] = _log(rng, 1, min(16384, int(math.sqrt(16384 * 16384 * 16 * 128 / (c["batch"] * c["heads"] * dim * (3 if c["type"] == "f32" else 1))))))
    if op == "decode":
        c["batch"] = _log(rng, 1, 128)
        c["tokens"] = _log(rng, 1, min(131072, 64 * 32768 * 8 * 128 // (c["batch"] * kv_heads * dim * (2 if c["type"] == "f32" else 1))))
    if op == "fork":
        c["branches"] = _log(rng, 2, 48)
        c["tokens"] = _log(rng, 5, 16384)
    if op == "turnover":
        c["sequences"], c["layers"] = 2 * rng.randint(1, 12), rng.randint(1, 4)
        c["tokens"] = _log(rng, 5, 4500)
    if op != "prompt":
        c["page"] = rng.choice([8, 16, 32, 64, 128])
    return c


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _lengths(case, seed):
    """Tokens of each sequence of a batch; a ragged one has lengths down to one token, and at least one whole sequence."""
    n, most = case["batch"], case["tokens"]
    if not case["ragged"]:
        return [most] * n
    rng = random.Random(seed)
    got = [max(1, int(round(most * rng.uniform(0.05, 1.0)))) for _ in range(n)]
    got[rng.randrange(n)] = most
    return got


def _values(case, seed, *shapes):
    """Normally distributed tensors, as projections of normalised positions are."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(s, generator=gen, device="cuda", dtype=torch.float32).to(TYPES[case["type"]]) for s in shapes]


def _pages(n, page):
    return -(-n // page)


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _cache(case, sequences, pages, heads, layers=1):
    import fyusenet_amd as fa
    return fa.SequenceCache(fa.STORAGE_F16 if case["type"] == "f16" else fa.STORAGE_F32, layers=layers, heads=heads, kv_heads=case["kv_heads"],
                            head_dim=case["dim"], page_tokens=case["page"], pages=pages, sequences=sequences)


def _pool(case, keys, values, offsets, lengths, pages, seed, shuffle):
    """A tensor of pages [page, keys or values, head, token, dim] with the tokens in it, and the sequences' lists of pages."""
    page, most = case["page"], _pages(max(lengths), case["page"])
    gen = torch.Generator().manual_seed(seed)
    order = torch.randperm(pages, generator=gen) if shuffle else torch.arange(pages)
    table, at = torch.zeros(len(lengths), most, dtype=torch.int64), 0
    for b, n in enumerate(lengths):
        table[b, :_pages(n, page)] = order[at:at + _pages(n, page)]
        at += _pages(n, page)
    table = table.cuda()
    pool = torch.zeros(pages, 2, case["kv_heads"], page, case["dim"], dtype=keys.dtype, device="cuda")
    for b, n in enumerate(lengths):
        t = torch.arange(n, device="cuda")
        pool[table[b, t // page], 0, :, t % page] = keys[offsets[b]:offsets[b] + n]
        pool[table[b, t // page], 1, :, t % page] = values[offsets[b]:offsets[b] + n]
    return pool, table


def prepare(case, seed):
    heads, kv, dim = case.get("heads"), case["kv_heads"], case["dim"]
    if case["op"] == "prompt":
        n, most = case["batch"], case["tokens"]
        q, k, v = _values(case, seed, (n, most, heads, dim), (n, most, kv, dim), (n, most, kv, dim))
        lengths = torch.tensor(_lengths(case, seed), dtype=torch.int32, device="cuda") if case["ragged"] else None
        return {"case": case, "q": q, "k": k, "v": v, "lengths": lengths, "out": torch.empty_like(q)}
    if case["op"] == "decode":
        lengths = _lengths(case, seed)
        total = sum(lengths)
        q, k, v = _values(case, seed, (case["batch"], heads, dim), (total, kv, dim), (total, kv, dim))
        pages = sum(_pages(n, case["page"]) for n in lengths) + 8
        state = {"case": case, "q": q, "out": torch.empty_like(q)}
        if own:
            # the sequences have grown side by side, so that their pages lie between each other's
            cache = _cache(case, case["batch"], pages, heads)
            for part in range(4):
                at = [(n * part // 4, n * (part + 1) // 4) for n in lengths]
                who = [b for b in range(len(lengths)) if at[b][1] > at[b][0]]
                if not who:
                    continue
                first = [sum(lengths[:b]) for b in who]
                rows = [slice(f + at[b][0], f + at[b][1]) for f, b in zip(first, who)]
                cache.extend(who, [at[b][1] - at[b][0] for b in who], stream=_stream())
                cache.write(0, torch.cat([k[r] for r in rows]), torch.cat([v[r] for r in rows]), stream=_stream())
            # the batch whose queries are asked for: one new token for each sequence
            cache.truncate(list(range(len(lengths))), [n - 1 for n in lengths], stream=_stream())
            cache.extend(list(range(len(lengths))), [1] * len(lengths), stream=_stream())
            last = torch.tensor([sum(lengths[:b + 1]) - 1 for b in range(len(lengths))], device="cuda")
            cache.write(0, k[last], v[last], stream=_stream())
            return dict(state, cache=cache)
        pool, table = _pool(case, k, v, [sum(lengths[:b]) for b in range(len(lengths))], lengths, pages, seed, True)
        return dict(state, pool=pool, table=table, lengths=torch.tensor(lengths, device="cuda"))
    if case["op"] == "fork":
        n, most, page = case["branches"], case["tokens"], case["page"]
        q, k, v, nk, nv = _values(case, seed, (n, heads, dim), (most, kv, dim), (most, kv, dim), (n, kv, dim), (n, kv, dim))
        state = {"case": case, "q": q, "nk": nk, "nv": nv, "out": torch.empty_like(q)}
        pages = _pages(most, page) + n + 8
        if own:
            cache = _cache(case, n + 1, pages, heads)
            cache.extend([0], [most], stream=_stream())
            cache.write(0, k, v, stream=_stream())
            return dict(state, cache=cache)
        pool, table = _pool(case, k, v, [0], [most], pages, seed, False)
        return dict(state, pool=pool, table=table[0], fresh=torch.arange(n, device="cuda") + _pages(most, page))
    # turnover
    n, most, page, layers = case["sequences"], case["tokens"], case["page"], case["layers"]
    k, v = _values(case, seed, (layers, n, most, kv, dim), (layers, n, most, kv, dim))
    state = {"case": case, "groups": (list(range(n // 2)), list(range(n // 2, n)))}
    if own:
        cache = _cache(case, n, n * _pages(most, page), kv, layers)
        cache.extend(list(range(n)), [most] * n, stream=_stream())
        for i in range(layers):
            cache.write(i, k[i].reshape(n * most, kv, dim), v[i].reshape(n * most, kv, dim), stream=_stream())
        return dict(state, cache=cache, keys=torch.empty_like(k), values=torch.empty_like(v))
    each = _pages(most, page)
    pool = torch.zeros(n, each, layers, 2, kv, page, dim, dtype=k.dtype, device="cuda")
    t = torch.arange(most, device="cuda")
    pool[:, t // page, :, 0, :, t % page] = k.permute(2, 1, 0, 3, 4)
    pool[:, t // page, :, 1, :, t % page] = v.permute(2, 1, 0, 3, 4)
    pool = pool.reshape(n * each, layers, 2, kv, page, dim)
    return dict(state, pool=pool, table=torch.arange(n * each, device="cuda").reshape(n, each))


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def _visible(case, i, j):
    see = j < j.shape[-1]
    if case.get("causal", True):
        see = see & (j <= i)
    if case.get("window", 0):
        see = see & (((i - j).abs() < case["window"]) | (j < case["sinks"]))
    return see


def _softmax_product(scores, see, values):
    """softmax over what is seen, times values; rows that see nothing are zero."""
    scores = scores.masked_fill(~see, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=torch.finfo(scores.dtype).min)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, values) / torch.where(total > 0, total, torch.ones_like(total))


def _plain_prompt(state):
    case = state["case"]
    n, most, heads, dim = state["q"].shape
    kv = case["kv_heads"]
    q = state["q"].float().permute(0, 2, 1, 3).reshape(n, kv, heads // kv * most, dim)
    k, v = (state[x].float().permute(0, 2, 1, 3) for x in "kv")
    at = torch.arange(most, device="cuda")
    see = _visible(case, at[:, None], at[None, :])
    if state["lengths"] is not None:
        inside = at[None, :] < state["lengths"][:, None]
        see = (see & inside[:, None, :] & inside[:, :, None])[:, None, None]
    scores = (torch.matmul(q, k.transpose(2, 3)) / math.sqrt(dim)).reshape(n, kv, heads // kv, most, most)
    out = _softmax_product(scores, see.expand(scores.shape), v[:, :, None].expand(-1, -1, heads // kv, -1, -1))
    return out.reshape(n, heads, most, dim).permute(0, 2, 1, 3).to(state["q"].dtype)


def _plain_step(case, q, pool, table, lengths):
    """One query per sequence: the last of `lengths` tokens, over the pages of `table`."""
    n, heads, dim = q.shape
    kv = case["kv_heads"]
    pages = pool[table].float()                                                     # [n, page, 2, kv, token, dim]
    k, v = (pages[:, :, x].permute(0, 2, 1, 3, 4).reshape(n, kv, -1, dim) for x in (0, 1))
    at = torch.arange(k.shape[2], device="cuda")
    see = (_visible(case, lengths[:, None] - 1, at[None, :]) & (at[None, :] < lengths[:, None]))[:, None, None, :]
    scores = torch.matmul(q.float().reshape(n, kv, heads // kv, dim), k.transpose(2, 3)) / math.sqrt(dim)
    return _softmax_product(scores, see, v).reshape(n, heads, dim).to(q.dtype)


def _plain_fork(state):
    case, pool, table, fresh = state["case"], state["pool"], state["table"], state["fresh"]
    n, most, page = case["branches"], case["tokens"], case["page"]
    lists = table.expand(n, -1)
    if most % page:
        pool[fresh] = pool[table[-1:]]                                              # a page that is written belongs to one branch
        lists = torch.cat([lists[:, :-1], fresh[:, None]], 1)
    else:
        lists = torch.cat([lists, fresh[:, None]], 1)
    pool[fresh, 0, :, most % page] = state["nk"]
    pool[fresh, 1, :, most % page] = state["nv"]
    return _plain_step(case, state["q"], pool, lists, torch.full((n,), most + 1, device="cuda"))


def _plain_turnover(state):
    case, pool, table = state["case"], state["pool"], state["table"]
    n, most, page, layers = case["sequences"], case["tokens"], case["page"], case["layers"]
    gone, stay = state["groups"]
    half = pool.shape[0] // 2
    pool[:half] = pool[half:]                                                       # those that stay lie in the upper half
    pool[half:] = pool[:half]
    low = torch.arange(half, device="cuda").reshape(n // 2, -1)
    table[stay], table[gone] = low, low + half
    state["groups"] = (stay, gone)
    got = pool[table].permute(3, 2, 0, 1, 5, 4, 6).reshape(2, layers, n, -1, case["kv_heads"], case["dim"])[:, :, :, :most]
    return {"keys": got[0].contiguous(), "values": got[1].contiguous()}


def run(state):
    case = state["case"]
    if not own:
        if case["op"] == "prompt":
            return _plain_prompt(state)
        if case["op"] == "decode":
            return _plain_step(case, state["q"], state["pool"], state["table"], state["lengths"])
        return _plain_fork(state) if case["op"] == "fork" else _plain_turnover(state)
    stream = _stream()
    if case["op"] == "prompt":
        import fyusenet_amd as fa
        fa.attention(state["q"], state["k"], state["v"], state["out"], lengths=state["lengths"], causal=case["causal"], window=case["window"],
                     sinks=case["sinks"], stream=stream)
        return state["out"]
    cache = state["cache"]
    if case["op"] == "decode":
        cache.attend(0, state["q"], state["out"], window=case["window"], sinks=case["sinks"], stream=stream)
        return state["out"]
    if case["op"] == "fork":
        branches = list(range(1, case["branches"] + 1))
        cache.fork(0, branches, stream=stream)
        cache.extend(branches, [1] * len(branches), stream=stream)
        cache.write(0, state["nk"], state["nv"], stream=stream)
        cache.attend(0, state["q"], state["out"], stream=stream)
        cache.free(branches, stream=stream)
        return state["out"]
    gone, stay = state["groups"]
    cache.free(gone, stream=stream)
    cache.compact(stream=stream)
    cache.copy(stay, gone, stream=stream)
    state["groups"] = (stay, gone)
    n, most = case["sequences"], case["tokens"]
    for i in range(case["layers"]):
        cache.read(list(range(n)), i, state["keys"][i].view(n * most, *state["keys"].shape[3:]), state["values"][i].view(n * most, *state["keys"].shape[3:]),
                   stream=stream)
    return {"keys": state["keys"], "values": state["values"]}


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without, and what it gives in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def _seen(case, i, n):
    """How many of the n tokens position i sees."""
    last = i + 1 if case.get("causal", True) else n
    w = case.get("window", 0)
    if not w:
        return last
    low, high = max(0, i - w + 1), min(last, i + w)
    return high - low + min(case["sinks"], low) + (max(0, min(case["sinks"], last) - high) if high < last else 0)


def work(case):
    size, kv, dim = (2 if case["type"] == "f16" else 4), case["kv_heads"], case["dim"]
    if case["op"] == "turnover":
        whole = case["sequences"] * case["tokens"] * case["layers"] * kv * dim * 2 * size
        return {"bytes": 2.5 * whole, "flops": 0}
    heads = case["heads"]
    if case["op"] == "fork":
        n, most = case["branches"], case["tokens"]
        tail = 2 * (most % case["page"]) * kv * dim * 2 * size * n
        return {"bytes": most * kv * dim * 2 * size + tail + n * (2 * heads + 4 * kv) * dim * size, "flops": 4.0 * n * heads * dim * (most + 1)}
    lengths = _lengths(case, 1)
    if case["op"] == "decode":
        seen = [_seen(case, n - 1, n) for n in lengths]
        return {"bytes": (sum(seen) * kv * 2 + 2 * len(lengths) * heads) * dim * size, "flops": 4.0 * heads * dim * sum(seen)}
    pairs = sum(sum(_seen(case, i, n) for i in range(n)) for n in lengths)
    return {"bytes": (sum(lengths) * (heads + 2 * kv) + case["batch"] * case["tokens"] * heads) * dim * size, "flops": 4.0 * heads * dim * pairs}


def _exact_attention(case, q, k, v, first):
    """q [m, heads, dim] are the tokens first..first+m-1 of a sequence k, v [n, kv_heads, dim]; head by head, in 64 bits."""
    m, heads, dim = q.shape
    n, group = k.shape[0], heads // case["kv_heads"]
    i, j = torch.arange(first, first + m, device="cuda")[:, None], torch.arange(n, device="cuda")[None, :]
    hidden = torch.zeros(m, n, dtype=torch.bool, device="cuda")
    if case.get("causal", True):
        hidden |= j > i
    if case.get("window", 0):
        hidden |= ((j <= i - case["window"]) | (j >= i + case["window"])) & (j >= case["sinks"])
    out = torch.zeros(m, heads, dim, dtype=torch.float64, device="cuda")
    for h in range(heads):
        s = (q[:, h].double() * dim ** -0.5) @ k[:, h // group].double().t()
        s[hidden] = -math.inf
        out[:, h] = torch.softmax(s, 1) @ v[:, h // group].double()
    return out


def exact(case, seed):
    heads, kv, dim = case.get("heads"), case["kv_heads"], case["dim"]
    if case["op"] == "prompt":
        n, most = case["batch"], case["tokens"]
        q, k, v = _values(case, seed, (n, most, heads, dim), (n, most, kv, dim), (n, most, kv, dim))
        out = torch.zeros(n, most, heads, dim, dtype=torch.float64, device="cuda")
        for b, m in enumerate(_lengths(case, seed)):
            out[b, :m] = _exact_attention(case, q[b, :m], k[b, :m], v[b, :m], 0)
        return out
    if case["op"] == "decode":
        lengths = _lengths(case, seed)
        q, k, v = _values(case, seed, (case["batch"], heads, dim), (sum(lengths), kv, dim), (sum(lengths), kv, dim))
        out, at = [], 0
        for b, m in enumerate(lengths):
            out.append(_exact_attention(case, q[b:b + 1], k[at:at + m], v[at:at + m], m - 1))
            at += m
        return torch.cat(out)
    if case["op"] == "fork":
        n, most = case["branches"], case["tokens"]
        q, k, v, nk, nv = _values(case, seed, (n, heads, dim), (most, kv, dim), (most, kv, dim), (n, kv, dim), (n, kv, dim))
        return torch.cat([_exact_attention(case, q[b:b + 1], torch.cat([k, nk[b:b + 1]]), torch.cat([v, nv[b:b + 1]]), most) for b in range(n)])
    n, most, layers = case["sequences"], case["tokens"], case["layers"]
    k, v = _values(case, seed, (layers, n, most, kv, dim), (layers, n, most, kv, dim))
    return {"keys": torch.cat([k[:, n // 2:]] * 2, 1).double(), "values": torch.cat([v[:, n // 2:]] * 2, 1).double()}
