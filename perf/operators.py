"""What a step of drafted tokens costs: the operators that verify a chain or a tree of drafts over the paged KV cache.

A serving program that drafts tokens runs, for a batch of sequences, one pass of its model over all drafted nodes at once:

  layout     once a step: ancestor masks and token positions of every node, from the trees' parents
  prologue   once a layer: head norm and RoPE at the nodes' positions, the query out, K and V into the pages
  attention  once a layer: every node attends to its sequence's cached tokens and to its own ancestors
  verify     once a step: accepts drafts against the target's probabilities from given random numbers, draws the next token
  commit     once a step: the accepted nodes' cache rows move behind the sequence's tokens, in every plane of every layer

Node 0 of a tree is the token that was sampled last; every other node's parent comes before it.  Node i of sequence b lies
at cache token kv_lens[b] + i.  `run` computes an operator from elementary torch operations, or calls the framework's own.
"""
from __future__ import annotations

import math

import torch

own = False

_DEV = "cuda"
_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_GOLDEN = 0.6180339887498949
_TREE, _CHAIN = "tree", "chain"


def listed():
    return [
        # one chat with a small draft tree: what a step pays before its first layer
        _layout(name="layout_step", batch=1, rows=8),
        # a batch of large trees of unequal sizes
        _layout(name="layout_batch", batch=64, rows=200, ragged=True),
        # one chat, a layer's norm, rotation and page writes of a small tree
        _prologue(name="prologue_step", batch=1, rows=8, heads=16, kv_heads=4, dim=128, context=4096),
        # the same for a serving batch of larger trees
        _prologue(name="prologue_batch", batch=32, rows=48, heads=64, kv_heads=8, dim=128, context=4096, ragged=True),
        # one chat, a short context, a small tree: latency
        _attention(name="attention_step_4k", batch=1, rows=7, heads=16, kv_heads=4, dim=128, context=4096),
        # a serving batch of long contexts, a chain of four drafts behind the sampled token
        _attention(name="attention_chain_32k", batch=8, rows=5, heads=64, kv_heads=8, dim=128, context=32768, shape=_CHAIN),
        # sequences of unequal lengths with trees of unequal sizes
        _attention(name="attention_tree_ragged", batch=8, rows=24, heads=32, kv_heads=8, dim=128, context=32768, ragged=True),
        # one long document with a wide tree
        _attention(name="attention_wide_50k", batch=1, rows=64, heads=64, kv_heads=8, dim=128, context=50000),
        # a sliding-window layer over f16 rows with a soft cap
        _attention(name="attention_f16_window", batch=4, rows=12, heads=16, kv_heads=8, dim=256, context=8192, cache="f16", window=1024, softcap=50.0),
        # one chat, a chain of four drafts with the draft model's distributions
        _verify(name="verify_step", batch=1, rows=5, vocab=32000, shape=_CHAIN),
        # a serving batch of trees over a large vocabulary, drafts without distributions
        _verify(name="verify_batch", batch=32, rows=32, vocab=130001, ragged=True),
        # the accepted rows of a batch, all layers at once
        _commit(name="commit_layers", batch=32, rows=24, heads=8, dim=128, layers=28, context=512),
    ]


def draw(rng):
    """Another case of the same ranges: sizes over their logarithm, and the options that occur with them."""
    kind = rng.choice(["layout", "prologue", "attention", "attention", "attention", "verify", "verify", "commit"])
    batch, rows = _log_int(rng, 1, 48), _log_int(rng, 2, 96)
    ragged = batch > 1 and rng.random() < 0.5
    shape = rng.choice([_TREE, _TREE, _CHAIN])
    page = rng.choice([16, 16, 32, 64, 24])
    if kind == "layout":
        return _layout(batch=_log_int(rng, 1, 64), rows=_log_int(rng, 2, 200), ragged=ragged)
    heads, kv_heads, dim, cache = rng.choice([(64, 8, 128, "q8"), (32, 8, 128, "q8"), (16, 4, 128, "q8"), (24, 8, 128, "q8"), (8, 1, 128, "q8"),
                                              (32, 8, 64, "q8"), (16, 2, 256, "q8"), (24, 4, 192, "q8"), (16, 8, 256, "f16"), (32, 8, 128, "f16")])
    if kind == "prologue":
        batch = min(batch, 32)
        return _prologue(batch=batch, rows=min(rows, 1536 // batch), heads=heads, kv_heads=kv_heads, dim=dim, cache=cache, context=_log_int(rng, 100, 4096),
                         ragged=ragged, page=page, layout=rng.choice(["half", "half", "interleaved"]), rotary=rng.choice([dim, dim, dim // 2]),
                         dtype=rng.choice(["bf16", "bf16", "f16", "f32"]))
    if kind == "attention":
        context = _log_int(rng, 64, 65536)
        row_bytes = _row_bytes(cache, kv_heads, dim)
        most = min(550e6 / (row_bytes * batch), 6.7e10 / (4.0 * dim * heads * batch * rows))
        context = max(16, min(context, int(most)))
        windowed = rng.random() < 0.3
        return _attention(batch=batch, rows=rows, heads=heads, kv_heads=kv_heads, dim=dim, context=context, cache=cache, ragged=ragged, shape=shape, page=page,
                          window=rng.choice([512, 1024]) if windowed else 0, softcap=50.0 if windowed else 0.0, dtype=rng.choice(["bf16", "bf16", "f16"]),
                          scales=rng.choice(["f16", "f16", "bf16"]))
    if kind == "verify":
        vocab = _log_int(rng, 1000, 200000)
        rows = max(2, min(rows, int(1.3e8 / (batch * vocab))))
        return _verify(batch=batch, rows=rows, vocab=vocab, shape=shape, ragged=ragged, dtype=rng.choice(["f32", "f32", "bf16"]))
    return _commit(batch=min(batch, 32), rows=rows, heads=kv_heads, dim=dim, layers=_log_int(rng, 1, 28), context=_log_int(rng, 64, 512), page=page, cache=cache)


def prepare(case, seed):
    gen = torch.Generator(device=_DEV)
    gen.manual_seed(seed)
    s = _PREPARE[case["kind"]](case, gen)
    s["case"] = case
    return s


def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["kind"]](state)


def work(case):
    """Every input read once and every output written once; multiply-adds of the (node, cached token) pairs."""
    kind, batch, rows = case["kind"], case["batch"], case["rows"]
    nodes = sum(_counts(case))
    if kind == "layout":
        return {"bytes": nodes * (4 + 8 * ((rows + 63) // 64) + 4) + 8 * batch, "flops": nodes * ((rows + 63) // 64)}
    if kind == "verify":
        rows_read = batch * (2 if case["shape"] == _CHAIN else 1)
        return {"bytes": rows_read * case["vocab"] * _size(case["dtype"]) + nodes * 20, "flops": 2 * rows_read * case["vocab"]}
    if kind == "commit":
        moved = sum(min(_accepted(n), n) - 1 for n in _counts(case))
        return {"bytes": max(2 * moved * case["layers"] * _row_bytes(case["cache"], case["heads"], case["dim"]), 8 * nodes), "flops": 0}
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    size, row_bytes = _size(case["dtype"]), _row_bytes(case["cache"], kv_heads, dim)
    if kind == "prologue":
        return {"bytes": nodes * ((2 * heads + 2 * kv_heads) * dim * size + row_bytes + 4 * case["rotary"]), "flops": 9 * nodes * (heads + 2 * kv_heads) * dim}
    keys = [min(n, case["window"] - 1) if case["window"] else n for n in _lengths(case)]
    pairs = sum((n + 1) * k for n, k in zip(keys, _counts(case)))
    return {"bytes": sum(n + k for n, k in zip(keys, _counts(case))) * row_bytes + 2 * nodes * heads * dim * size, "flops": 4 * dim * heads * pairs}


def exact(case, seed):
    """The operators' definitions in 64 bits, one sequence (and one head, one node) at a time."""
    s = prepare(case, seed)
    return {"layout": _none, "prologue": _exact_prologue, "attention": _exact_attention, "verify": _none, "commit": _none}[case["kind"]](s)


# ---- cases --------------------------------------------------------------------------------------------------------------


def _layout(batch, rows, ragged=False, name=None):
    return _named(name, kind="layout", batch=batch, rows=rows, ragged=ragged)


def _prologue(batch, rows, heads, kv_heads, dim, context, cache="q8", ragged=False, page=16, layout="half", rotary=None, dtype="bf16", name=None):
    return _named(name, kind="prologue", batch=batch, rows=rows, heads=heads, kv_heads=kv_heads, dim=dim, context=context, cache=cache, ragged=ragged, page=page,
                  layout=layout, rotary=dim if rotary is None else rotary, dtype=dtype)


def _attention(batch, rows, heads, kv_heads, dim, context, cache="q8", ragged=False, shape=_TREE, page=16, window=0, softcap=0.0, dtype="bf16", scales="f16",
               name=None):
    return _named(name, kind="attention", batch=batch, rows=rows, heads=heads, kv_heads=kv_heads, dim=dim, context=context, cache=cache, ragged=ragged,
                  shape=shape, page=page, window=window, softcap=softcap, dtype=dtype, scales=scales)


def _verify(batch, rows, vocab, shape=_TREE, ragged=False, dtype="f32", name=None):
    return _named(name, kind="verify", batch=batch, rows=rows, vocab=vocab, shape=shape, ragged=ragged, dtype=dtype)


def _commit(batch, rows, heads, dim, layers, context, page=16, cache="q8", name=None):
    return _named(name, kind="commit", batch=batch, rows=rows, heads=heads, dim=dim, layers=layers, context=context, page=page, cache=cache, ragged=False)


def _named(name, **case):
    return case if name is None else {"name": name, **case}


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _size(dtype):
    return 4 if dtype == "f32" else 2


def _row_bytes(cache, kv_heads, dim):
    return 4 * kv_heads * dim if cache == "f16" else 2 * (kv_heads * dim + kv_heads * dim // 64 * 2)


def _spread(low, high, i):
    return low + int((high - low) * ((i + 1) * _GOLDEN % 1.0))


def _lengths(case):
    """Cached tokens of each sequence: all `context`, or spread over [context / 32, context]."""
    context = case["context"]
    return [_spread(context // 32 + 1, context, i) if case["ragged"] else context for i in range(case["batch"])]


def _counts(case):
    """Nodes of each sequence's tree: all `rows`, or spread over [rows / 2, rows]."""
    rows = case["rows"]
    return [_spread((rows + 1) // 2, rows, 2 * i + 1) if case["ragged"] else rows for i in range(case["batch"])]


def _accepted(nodes):
    """Nodes of an accepted path: a few, the sampled token among them."""
    return max(1, min(nodes // 2, 5))


# ---- inputs -------------------------------------------------------------------------------------------------------------


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=_DEV)


def _randn(gen, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=gen, device=_DEV, dtype=dtype)


def _randint(gen, high, *shape):
    return torch.randint(0, high, shape, generator=gen, device=_DEV)


def _counts_tensor(case):
    return _ints(_counts(case)) if case["ragged"] else None


def _parents(case, gen):
    """Trees that grow near their newest nodes: a node's parent is one of the eight before it (a chain: the one before it)."""
    batch, rows = case["batch"], case["rows"]
    index = torch.arange(rows, device=_DEV)
    if case.get("shape") == _CHAIN:
        parents = (index - 1).expand(batch, rows)
    else:
        back = 1 + _randint(gen, 8, batch, rows)
        parents = torch.where(index > 0, (index - back).clamp(min=0), -1)
    return parents.to(torch.int32).contiguous()


def _ancestors(parents):
    """[batch, rows, rows] truth: node j is node i or an ancestor of it; and depths [batch, rows]."""
    batch, rows = parents.shape
    seen = torch.zeros(batch, rows, rows, dtype=torch.bool, device=_DEV)
    depth = torch.zeros(batch, rows, dtype=torch.int32, device=_DEV)
    at = torch.arange(batch, device=_DEV)
    for i in range(rows):
        parent = parents[:, i].long()
        has = parent >= 0
        parent = parent.clamp(min=0)
        seen[:, i] = seen[at, parent] & has[:, None]
        depth[:, i] = torch.where(has, depth[at, parent] + 1, 0)
        seen[:, i, i] = True
    return seen, depth


def _pack(seen):
    """Truth values [.., rows] as 64-bit words [.., ceil(rows / 64)], the first in the lowest bit."""
    rows = seen.shape[-1]
    words = (rows + 63) // 64
    bits = torch.zeros(*seen.shape[:-1], words * 64, dtype=torch.int64, device=_DEV)
    bits[..., :rows] = seen.to(torch.int64)
    return (bits.view(*seen.shape[:-1], words, 64) << torch.arange(64, device=_DEV)).sum(-1)


def _unpack(masks, rows):
    bits = (masks[..., None] >> torch.arange(64, device=_DEV)) & 1
    return bits.flatten(-2)[..., :rows].bool()


def _tables(gen, lengths, page):
    """Block tables [sequences, pages of the longest] and the pool's rows: pages in random order, without replacement."""
    pages = [(n + page - 1) // page for n in lengths]
    pool = sum(pages) + sum(pages) // 4 + 1
    order = torch.randperm(pool, generator=gen, device=_DEV).to(torch.int32)
    tables = torch.zeros(len(lengths), max(pages), dtype=torch.int32, device=_DEV)
    at = 0
    for b, n in enumerate(pages):
        tables[b, :n] = order[at : at + n]
        at += n
    return tables, pool * page


def _plane_pair(gen, rows, cols, cache, scales):
    """A pool of rows ~N(0, 1), 1 % of the channels eight times larger: f16 values, or int8 codes with a scale per 64 columns."""
    gain = torch.ones(cols, device=_DEV)
    gain[torch.randperm(cols, generator=gen, device=_DEV)[: max(1, cols // 100)]] = 8.0
    if cache == "f16":
        return (_randn(gen, rows, cols, dtype=torch.float16) * gain.half()), None
    codes = torch.empty(rows, cols, dtype=torch.int8, device=_DEV)
    steps = torch.empty(rows, cols // 64, dtype=torch.float16 if scales == "f16" else torch.bfloat16, device=_DEV)
    for at in range(0, rows, 65536):
        x = (_randn(gen, min(65536, rows - at), cols) * gain).view(-1, cols // 64, 64)
        step = x.abs().amax(-1) / 127.0
        steps[at : at + x.shape[0]] = step
        codes[at : at + x.shape[0]] = torch.round(x / step[..., None]).clamp(-127, 127).view(-1, cols)
    return codes, steps


def _cache(case, gen, lengths, kv_heads, scales="f16"):
    tables, rows = _tables(gen, lengths, case["page"])
    s = {"tables": tables}
    s["k"], s["k_scales"] = _plane_pair(gen, rows, kv_heads * case["dim"], case["cache"], scales)
    s["v"], s["v_scales"] = _plane_pair(gen, rows, kv_heads * case["dim"], case["cache"], scales)
    return s


def _prepare_layout(case, gen):
    return {"parents": _parents(case, gen), "kv_lens": 1 + _randint(gen, 30000, case["batch"]).to(torch.int32), "counts": _counts_tensor(case)}


def _prepare_prologue(case, gen):
    batch, rows, dim, dtype = case["batch"], case["rows"], case["dim"], _DTYPES[case["dtype"]]
    lengths = _lengths(case)
    s = _cache(case, gen, [n + rows for n in lengths], case["kv_heads"])
    s.update(kv_lens=_ints(lengths), counts=_counts_tensor(case))
    _, depth = _ancestors(_parents(case, gen))
    s["positions"] = s["kv_lens"][:, None] + depth
    s["q"] = _randn(gen, batch * rows, case["heads"] * dim).to(dtype)
    for name in ("k_new", "v_new"):
        s[name] = _randn(gen, batch * rows, case["kv_heads"] * dim).to(dtype)
    s["q_norm"], s["k_norm"] = _randn(gen, dim) * 0.1, _randn(gen, dim) * 0.1
    half = case["rotary"] // 2
    angle = torch.arange(case["context"] + rows, device=_DEV, dtype=torch.float64)[:, None] / 10000.0 ** (torch.arange(half, device=_DEV, dtype=torch.float64) / half)
    s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    return s


def _prepare_attention(case, gen):
    batch, rows = case["batch"], case["rows"]
    lengths = _lengths(case)
    s = _cache(case, gen, [n + rows for n in lengths], case["kv_heads"], case["scales"])
    seen, depth = _ancestors(_parents(case, gen))
    s.update(kv_lens=_ints(lengths), counts=_counts_tensor(case), masks=_pack(seen))
    s["positions"] = s["kv_lens"][:, None] + depth
    s["q"] = _randn(gen, batch * rows, case["heads"] * case["dim"]).to(_DTYPES[case["dtype"]])
    s["longest"], s["total"] = max(lengths), sum(lengths)
    return s


def _prepare_verify(case, gen):
    """Peaked target distributions; a chain's drafts come from distributions near the target's, a tree's are its likeliest tokens."""
    batch, rows, vocab, dtype = case["batch"], case["rows"], case["vocab"], _DTYPES[case["dtype"]]
    parents = _parents(case, gen)
    hot = _randint(gen, vocab, batch, rows, 4)
    boost = torch.tensor([0.0, -0.5, -1.0, -1.5], device=_DEV) + math.log(vocab) + 3.0
    target = torch.empty(batch, rows, vocab, dtype=dtype, device=_DEV)
    drafts = torch.empty(batch, rows - 1, vocab, dtype=dtype, device=_DEV) if case["shape"] == _CHAIN else None
    tokens = torch.empty(batch, rows, dtype=torch.int64, device=_DEV)
    tokens[:, 0] = _randint(gen, vocab, batch)
    for b in range(batch):
        logits = _randn(gen, rows, vocab).scatter_(1, hot[b], boost.expand(rows, 4))
        target[b] = torch.softmax(logits, -1).to(dtype)
        if drafts is not None:
            q = torch.softmax(logits[:-1] + 0.5 * _randn(gen, rows - 1, vocab), -1).to(dtype)
            drafts[b] = q
            pick = torch.rand(rows - 1, 1, generator=gen, device=_DEV, dtype=torch.float64) * 0.999
            tokens[b, 1:] = torch.searchsorted(torch.cumsum(q.double(), -1), pick, right=True)[:, 0].clamp(max=vocab - 1)
        else:
            parent = parents[b, 1:].long()
            tokens[b, 1:] = hot[b][parent, _randint(gen, 4, rows - 1)]
    s = {"tokens": tokens.to(torch.int32), "parents": None if case["shape"] == _CHAIN else parents, "target": target, "drafts": drafts}
    s["uniforms"] = torch.rand(batch, rows, generator=gen, device=_DEV)
    s["counts"] = _counts_tensor(case)
    return s


def _prepare_commit(case, gen):
    """Accepted paths whose rows, but for the first, lie behind the places they move to: a pass can then be repeated."""
    batch, rows, cols, layers = case["batch"], case["rows"], case["heads"] * case["dim"], case["layers"]
    lengths = [_spread(case["context"] // 4, case["context"], i) for i in range(batch)]
    tables, pool = _tables(gen, [n + rows for n in lengths], case["page"])
    s = {"tables": tables, "kv_lens": _ints(lengths)}
    names = ("k", "v") if case["cache"] == "f16" else ("k", "k_scales", "v", "v_scales")
    for name in names:
        if case["cache"] == "f16":
            s[name] = _randn(gen, layers, pool, cols, dtype=torch.float16)
        elif name.endswith("scales"):
            s[name] = torch.rand(layers, pool, cols // 64, generator=gen, device=_DEV).half()
        else:
            s[name] = torch.randint(-127, 128, (layers, pool, cols), generator=gen, device=_DEV, dtype=torch.int8)
    s["names"] = names
    path = torch.full((batch, rows), -1, dtype=torch.int32)
    most = _accepted(rows)
    taken = _randint(gen, most, batch).tolist()
    spots = torch.rand(batch, rows, generator=gen, device=_DEV).cpu()
    for b in range(batch):
        count = taken[b] + 1
        path[b, 0] = 0
        free = torch.arange(count, rows)
        path[b, 1:count] = free[spots[b, : len(free)].argsort()[: count - 1]].sort().values.to(torch.int32)
    s["path"], s["accepted"] = path.to(_DEV), _ints([t + 1 for t in taken])
    s["planes"] = [s[name][layer] for layer in range(layers) for name in names]
    if own:
        from zllm_amd import ops

        s["plane_list"] = ops.commit_planes(s["planes"])
    return s


# ---- plain forms --------------------------------------------------------------------------------------------------------


def _live(s, batch, rows):
    """[batch, rows] truth: node i of sequence b is there."""
    if s["counts"] is None:
        return torch.ones(batch, rows, dtype=torch.bool, device=_DEV)
    return torch.arange(rows, device=_DEV) < s["counts"][:, None]


def _plain_layout(s):
    """A node sees itself and what its parent sees, one deeper; nodes that are not there see nothing and keep the sequence's length."""
    seen, depth = _ancestors(s["parents"])
    live = _live(s, *s["parents"].shape)
    return {"masks": _pack(seen & live[..., None]), "positions": s["kv_lens"][:, None] + torch.where(live, depth, 0).to(torch.int32)}


def _norm_rows(x, weight):
    """x * (1 / sqrt(mean of squares + eps)) * (1 + weight); eight running sums of every eighth square, then added in pairs."""
    squares = x.view(*x.shape[:-1], -1, 8)
    total = torch.zeros_like(squares[..., 0, :])
    for c in range(squares.shape[-2]):
        total = total + squares[..., c, :] * squares[..., c, :]
    total = total[..., :4] + total[..., 4:]
    total = total[..., :2] + total[..., 2:]
    total = total[..., :1] + total[..., 1:]
    inverse = 1.0 / torch.sqrt(total / float(x.shape[-1]) + 1e-6)
    return x * inverse * (weight + 1.0)


def _rotate(x, cos, sin, layout):
    """Pairs (i, i + half) or (2 i, 2 i + 1) of the first columns turned by the row's angles; the other columns stay."""
    half = cos.shape[-1]
    cos, sin = cos[:, None], sin[:, None]
    turned, rest = x[..., : 2 * half], x[..., 2 * half :]
    if layout == "half":
        a, b = turned[..., :half], turned[..., half:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)
    a, b = turned[..., 0::2], turned[..., 1::2]
    return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), rest], -1)


def _slots(s, case):
    """Physical cache row of every node [batch * rows]."""
    batch, rows, page = case["batch"], case["rows"], case["page"]
    token = s["kv_lens"].long()[:, None] + torch.arange(rows, device=_DEV)
    return (torch.gather(s["tables"].long(), 1, token // page) * page + token % page).flatten()


def _plain_prologue(s):
    case = s["case"]
    batch, rows, dim = case["batch"], case["rows"], case["dim"]
    live = _live(s, batch, rows).flatten()
    at = s["positions"].flatten().long()
    cos, sin = s["cos"][at], s["sin"][at]
    q = _rotate(_norm_rows(s["q"].float().view(-1, case["heads"], dim), s["q_norm"]), cos, sin, case["layout"])
    k = _rotate(_norm_rows(s["k_new"].float().view(-1, case["kv_heads"], dim), s["k_norm"]), cos, sin, case["layout"])
    v = s["v_new"].float().view(-1, case["kv_heads"], dim)
    out_dtype = torch.float32 if case["dtype"] == "f32" else _DTYPES[case["dtype"]]
    q = torch.where(live[:, None, None], q, 0.0).to(out_dtype).view(batch * rows, -1)
    slots = _slots(s, case)[live]
    result = {"q": q}
    for name, x in (("k", k), ("v", v)):
        x = x.reshape(batch * rows, -1)[live]
        if case["cache"] == "f16":
            s[name][slots] = x.half()
        else:
            groups = x.view(x.shape[0], -1, 64)
            most = groups.abs().amax(-1)
            step = torch.where(most > 0, most / 127.0, 1.0)
            s[name][slots] = torch.round(groups * (1.0 / step)[..., None]).clamp(-127, 127).to(torch.int8).view(x.shape)
            s[name + "_scales"][slots] = step.half()
            result[name + "_scales"] = s[name + "_scales"]
        result[name] = s[name]
    return result


def _rows_f32(s, name, physical, case):
    x = s[name][physical].float()
    if case["cache"] != "f16":
        x = (x.view(x.shape[0], -1, 64) * s[name + "_scales"][physical].float()[..., None]).view(x.shape[0], -1)
    return x.view(x.shape[0], case["kv_heads"], case["dim"])


def _plain_attention(s):
    case = s["case"]
    batch, rows, heads, kv_heads, dim, page, window = (case[k] for k in ("batch", "rows", "heads", "kv_heads", "dim", "page", "window"))
    seen = _unpack(s["masks"], rows)
    lengths, counts = _lengths(case), _counts(case)
    out = torch.zeros(batch, rows, heads, dim, device=_DEV)
    for b in range(batch):
        n, count = lengths[b], counts[b]
        first = max(0, n + 1 - window) if window else 0
        token = torch.arange(first, n + count, device=_DEV)
        physical = s["tables"][b].long()[token // page] * page + token % page
        k, v = _rows_f32(s, "k", physical, case), _rows_f32(s, "v", physical, case)
        position = s["positions"][b, :count]
        at = torch.cat([token[: n - first], position])
        visible = torch.cat([torch.ones(count, n - first, dtype=torch.bool, device=_DEV), seen[b, :count, :count]], 1)
        if window:
            visible = visible & (at[None, :] + window > position[:, None])
        q = s["q"].view(batch, rows, kv_heads, heads // kv_heads, dim)[b, :count].float()
        for h in range(kv_heads):
            score = (q[:, h].reshape(-1, dim) @ k[:, h].T.contiguous()) * dim**-0.5
            if case["softcap"]:
                score = case["softcap"] * torch.tanh(score / case["softcap"])
            score = torch.where(visible.repeat_interleave(heads // kv_heads, 0), score, -math.inf)
            weight = torch.exp(score - score.amax(-1, keepdim=True))
            mixed = (weight @ v[:, h].contiguous()) / weight.sum(-1, keepdim=True)
            out[b, :count, h * (heads // kv_heads) : (h + 1) * (heads // kv_heads)] = mixed.view(count, heads // kv_heads, dim)
    return out.view(batch * rows, heads * dim).to(s["q"].dtype)


def _plain_verify(s):
    """Walks all trees of the batch node by node; probabilities, their differences and sums in 64 bits, compared as they are."""
    tokens, target, uniforms = s["tokens"].long(), s["target"], s["uniforms"].double()
    batch, rows, vocab = target.shape
    live = _live(s, batch, rows)
    index = torch.arange(rows, device=_DEV)
    parents = (s["parents"] if s["parents"] is not None else (index - 1).expand(batch, rows)).long()
    at = torch.arange(batch, device=_DEV)
    p = target[at[:, None], parents.clamp(min=0), tokens].double()
    same = (tokens[:, :, None] == tokens[:, None, :]) & (parents[:, :, None] == parents[:, None, :]) & (index[:, None] > index[None, :])
    p = torch.where(same.any(-1), 0.0, p)
    q = s["drafts"][at[:, None], (index - 1).clamp(min=0), tokens].double() if s["drafts"] is not None else None
    current = torch.zeros(batch, dtype=torch.int64, device=_DEV)
    left = torch.ones(batch, dtype=torch.float64, device=_DEV)
    taken = torch.zeros(batch, rows, dtype=torch.bool, device=_DEV)
    taken[:, 0] = True
    for i in range(1, rows):
        child = (parents[:, i] == current) & live[:, i]
        accept = child & (uniforms[:, i] * (left if q is None else q[:, i]) < p[:, i])
        left = torch.where(accept, 1.0, torch.where(child, left - p[:, i], left))
        current = torch.where(accept, i, current)
        taken[:, i] = accept
    row = target[at, current].double()
    if q is not None:
        behind = current + 1
        rejected = (behind < rows) & live[at, behind.clamp(max=rows - 1)]
        weight = torch.where(rejected[:, None], (row - s["drafts"][at, current.clamp(max=rows - 2)].double()).clamp(min=0), row)
    else:
        weight = row.clone()
        struck = (parents == current[:, None]) & live & (index > 0)
        weight[at[:, None].expand(batch, rows)[struck], tokens[struck]] = 0.0
    weight = torch.where(weight.sum(-1, keepdim=True) > 0, weight, row)
    running = torch.cumsum(weight, -1)
    pick = (running <= uniforms[:, :1] * running[:, -1:]).sum(-1).clamp(max=vocab - 1)
    count = taken.sum(-1)
    path = torch.where(taken, index, rows).sort(-1).values
    path = torch.where(path < rows, path, -1)
    following = torch.gather(tokens, 1, path.roll(-1, 1).clamp(min=0))
    out = torch.where(index < count[:, None] - 1, following, -1)
    out = torch.where(index == count[:, None] - 1, pick[:, None], out)
    return {"path": path.to(torch.int32), "accepted": count.to(torch.int32), "tokens": out.to(torch.int32)}


def _plain_commit(s):
    case = s["case"]
    batch, rows, page = case["batch"], case["rows"], case["page"]
    index = torch.arange(rows, device=_DEV)
    move = index < s["accepted"][:, None]
    base = s["kv_lens"].long()[:, None]
    source, goal = base + s["path"].long().clamp(min=0), base + index
    tables = s["tables"].long()
    source = (torch.gather(tables, 1, source // page) * page + source % page)[move]
    goal = (torch.gather(tables, 1, goal // page) * page + goal % page)[move]
    for name in s["names"]:
        s[name][:, goal] = s[name][:, source]
    return {"lens": s["kv_lens"] + s["accepted"], **{name: s[name] for name in s["names"]}}


# ---- the framework's operators ------------------------------------------------------------------------------------------


def _own_layout(s):
    from zllm_amd import ops

    masks, positions = ops.draft_layout(s["parents"], s["kv_lens"], row_counts=s["counts"])
    return {"masks": masks, "positions": positions}


def _own_prologue(s):
    from zllm_amd import capi, ops

    case = s["case"]
    f16 = case["cache"] == "f16"
    q = ops.gqa_draft_prologue(s["q"], s["k_new"], s["v_new"], s["q_norm"], s["k_norm"], s["cos"], s["sin"], s["k"], s["k_scales"], s["v"], s["v_scales"],
                               s["tables"], s["kv_lens"], case["heads"], case["kv_heads"], case["dim"], case["rotary"], case["page"], positions=s["positions"],
                               row_counts=s["counts"], split_half=case["layout"] == "half", q_out_dtype=_DTYPES[case["dtype"]],
                               kv_format=capi.KV_F16 if f16 else capi.KV_Q8G64)
    return {"q": q, "k": s["k"], "v": s["v"]} if f16 else {"q": q, "k": s["k"], "k_scales": s["k_scales"], "v": s["v"], "v_scales": s["v_scales"]}


def _own_attention(s):
    from zllm_amd import capi, ops

    case = s["case"]
    return ops.gqa_draft_attention(s["q"], s["k"], s["k_scales"], s["v"], s["v_scales"], s["tables"], s["kv_lens"], s["masks"], case["heads"], case["kv_heads"],
                                   case["dim"], case["page"], case["dim"] ** -0.5, s["longest"], positions=s["positions"], row_counts=s["counts"],
                                   window=case["window"], softcap=case["softcap"], kv_format=capi.KV_F16 if case["cache"] == "f16" else capi.KV_Q8G64,
                                   scale_dtype=capi.SCALE_F16 if case["scales"] == "f16" else capi.SCALE_BF16, out_dtype=s["q"].dtype,
                                   total_kv_tokens=s["total"])


def _own_verify(s):
    from zllm_amd import ops

    path, accepted, tokens = ops.draft_verify(s["tokens"], s["target"], s["uniforms"], parents=s["parents"], draft_probs=s["drafts"], row_counts=s["counts"])
    return {"path": path, "accepted": accepted, "tokens": tokens}


def _own_commit(s):
    from zllm_amd import ops

    lens = ops.commit_rows(s["plane_list"], s["tables"], s["kv_lens"], s["path"], s["accepted"], s["case"]["page"])
    return {"lens": lens, **{name: s[name] for name in s["names"]}}


# ---- 64 bits ------------------------------------------------------------------------------------------------------------


def _none(s):
    return None


def _exact_prologue(s):
    case = s["case"]
    batch, rows, heads, dim, half = case["batch"], case["rows"], case["heads"], case["dim"], case["rotary"] // 2
    x = s["q"].double().view(batch, rows, heads, dim)
    x = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-6) * (1.0 + s["q_norm"].double())
    where = s["positions"].long()
    turn = torch.complex(s["cos"].double()[where], s["sin"].double()[where])[:, :, None]
    head = x[..., : 2 * half]
    pairs = torch.complex(head[..., :half].contiguous(), head[..., half:].contiguous()) if case["layout"] == "half" else torch.view_as_complex(head.reshape(batch, rows, heads, half, 2).contiguous())
    pairs = torch.view_as_real(pairs * turn)
    x[..., : 2 * half] = torch.cat([pairs[..., 0], pairs[..., 1]], -1) if case["layout"] == "half" else pairs.flatten(-2)
    for b, count in enumerate(_counts(case)):
        x[b, count:] = 0.0
    result = {"q": x.view(batch * rows, -1), "k": None, "v": None}
    if case["cache"] != "f16":
        result.update(k_scales=None, v_scales=None)
    return result


def _exact_attention(s):
    """Keys in blocks of 4096 with running maxima and sums, every head on its own."""
    case = s["case"]
    batch, rows, heads, dim, page = (case[k] for k in ("batch", "rows", "heads", "dim", "page"))
    group, wide = heads // case["kv_heads"], case["window"] or 1 << 40
    q = s["q"].double().view(batch, rows, heads, dim)
    out = torch.zeros(batch, rows, heads, dim, dtype=torch.float64, device=_DEV)
    bit = torch.arange(rows, device=_DEV)
    for b, (n, count) in enumerate(zip(_lengths(case), _counts(case))):
        own_position = s["positions"][b].long()
        for h0 in range(0, heads, group):
            columns = slice(h0 // group * dim, (h0 // group + 1) * dim)
            query = q[b, :count, h0 : h0 + group].reshape(count * group, dim)
            top = torch.full((count * group, 1), -math.inf, dtype=torch.float64, device=_DEV)
            total, mixed = torch.zeros_like(top), torch.zeros(count * group, dim, dtype=torch.float64, device=_DEV)
            for begin in range(max(0, n + 1 - wide) // 4096 * 4096, n + count, 4096):
                token = torch.arange(begin, min(begin + 4096, n + count), device=_DEV)
                row = s["tables"][b].long()[token // page] * page + token % page
                kv = []
                for name in ("k", "v"):
                    x = s[name][row, columns].double()
                    if case["cache"] != "f16":
                        x = x * s[name + "_scales"][row].double().repeat_interleave(64, 1)[:, columns]
                    kv.append(x)
                node = (token - n).clamp(0, rows - 1)
                where = torch.where(token < n, token, own_position[node])
                mask = s["masks"][b, :count][:, node // 64] >> (node % 64) & 1
                sees = ((token < n) | (mask == 1)) & (where + wide > own_position[:count, None])
                logit = torch.matmul(query, kv[0].T.contiguous()) / math.sqrt(dim)
                if case["softcap"]:
                    logit = case["softcap"] * torch.tanh(logit / case["softcap"])
                logit = logit.masked_fill(~sees.repeat_interleave(group, 0), -math.inf)
                new = torch.maximum(top, logit.amax(-1, keepdim=True))
                safe = torch.where(torch.isinf(new), 0.0, new)
                part, keep = torch.exp(logit - safe), torch.exp(top - safe)
                total, mixed, top = total * keep + part.sum(-1, keepdim=True), mixed * keep + torch.matmul(part, kv[1]), new
            out[b, :count, h0 : h0 + group] = (mixed / total).view(count, group, dim)
    return out.view(batch * rows, heads * dim)


_PREPARE = {"layout": _prepare_layout, "prologue": _prepare_prologue, "attention": _prepare_attention, "verify": _prepare_verify, "commit": _prepare_commit}
_PLAIN = {"layout": _plain_layout, "prologue": _plain_prologue, "attention": _plain_attention, "verify": _plain_verify, "commit": _plain_commit}
_OWN = {"layout": _own_layout, "prologue": _own_prologue, "attention": _own_attention, "verify": _own_verify, "commit": _own_commit}
