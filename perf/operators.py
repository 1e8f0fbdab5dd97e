"""Workloads of the attention operators for sequences of different lengths: packed prompts and a paged cache.

Three operators, as a program that trains on packed texts or serves a language model calls them:

* ``packed``: causal attention over sequences of different lengths that lie one behind the other in
  ``[tokens, heads, headdim]`` tensors, with fewer key and value heads than query heads
  (:func:`flash_attention_packed`); ``direction`` is ``forward`` (scoring, prefilling) or ``train`` (with its gradients);
* ``append``: keys and values of new tokens written into the pages of a cache, the position rotation of keys and
  queries applied on the way (:func:`append_kv_cache`): one new token a sequence, or the tokens of whole prompts;
* ``decode``: attention of one new token a sequence over its pages of that cache (:func:`flash_attention_decode`).

``run`` computes them with elementary torch operations in 32 bits, or, where ``own`` is true, with the package's kernels.
A case holds ``batch`` sequences whose lengths lie between ``low`` and ``high`` (spread over their logarithm, drawn
from ``salt``; the seed of ``prepare`` changes their order), ``heads`` and ``kv_heads``, ``headdim``, ``dtype``, and

* ``packed``: ``layout``: ``dense`` (three tensors) or ``fused`` (one ``[tokens, heads + 2 kv_heads, headdim]``
  projection), ``behind``: rows behind the last sequence (a buffer of fixed size);
* ``append``: ``fresh``: whether the tokens are whole prompts (``prompt``) or one a sequence (``token``),
  ``rotary``: how many columns are rotated (0: none), ``interleaved``: pairs of adjacent columns or of two halves,
  ``page``: tokens a page;
* ``decode``: ``page``.
"""

from __future__ import annotations

import math
import random

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
#: what the largest listed cases cost: score elements of the padded batch and multiply-adds times two (packed),
#: elements of keys in the cache (append and decode), elements of new keys (append)
_MOST_SCORES = 3 * 16 * 8192 * 8192
_MOST_TOKENS = 65536
_MOST_CACHE = 128 * 8192 * 8 * 128
_MOST_FRESH = 32768 * 8 * 128


def _packed(name, direction, batch, low, high, heads, kv_heads, headdim, dtype, layout="dense", behind=0, salt=1):
    return {"name": name, "op": "packed", "direction": direction, "batch": batch, "low": low, "high": high,
            "heads": heads, "kv_heads": kv_heads, "headdim": headdim, "dtype": dtype, "layout": layout,
            "behind": behind, "salt": salt}


def _append(name, fresh, batch, low, high, heads, kv_heads, headdim, dtype, page, rotary, interleaved=False, salt=1):
    return {"name": name, "op": "append", "fresh": fresh, "batch": batch, "low": low, "high": high, "heads": heads,
            "kv_heads": kv_heads, "headdim": headdim, "dtype": dtype, "page": page, "rotary": rotary,
            "interleaved": interleaved, "salt": salt}


def _decode(name, batch, low, high, heads, kv_heads, headdim, dtype, page, salt=1):
    return {"name": name, "op": "decode", "batch": batch, "low": low, "high": high, "heads": heads,
            "kv_heads": kv_heads, "headdim": headdim, "dtype": dtype, "page": page, "salt": salt}


def listed():
    return [
        # a handful of short questions scored in one call: the time of a call
        _packed("packed_short", "forward", 4, 16, 128, 8, 2, 64, "bf16"),
        # prefilling the prompts that came in together, projections fused as one tensor
        _packed("packed_prefill", "forward", 6, 256, 4096, 32, 8, 128, "bf16", layout="fused"),
        # training a small model on packed texts in a buffer of fixed size
        _packed("packed_train", "train", 8, 256, 1024, 16, 4, 64, "fp16", behind=100),
        # training on long documents
        _packed("packed_train_long", "train", 3, 4096, 8192, 16, 4, 128, "bf16"),
        # one decoding step of a few conversations: the time of a call
        _append("append_few", "token", 4, 100, 1000, 8, 2, 64, "bf16", 16, 64),
        # one decoding step of a full server
        _append("append_step", "token", 256, 200, 4000, 32, 8, 128, "bf16", 16, 128),
        # prompts whose projections go into the cache and on to attention, half of the columns rotated in adjacent pairs
        _append("append_prompts_pairs", "prompt", 12, 100, 3000, 16, 4, 80, "fp16", 24, 32, interleaved=True),
        # the prompts of a full server
        _append("append_prompts", "prompt", 16, 700, 4096, 32, 8, 128, "bf16", 64, 128),
        # one conversation
        _decode("decode_one", 1, 900, 900, 8, 2, 64, "bf16", 16),
        # a few very long contexts, heads of one GPU of a tensor-parallel group
        _decode("decode_long", 2, 100000, 131072, 16, 2, 128, "bf16", 64),
        # narrow heads, each with its own keys, pages of odd size
        _decode("decode_heads", 32, 100, 2000, 12, 12, 64, "fp16", 24),
        # a full server: many sequences of all lengths
        _decode("decode_server", 128, 500, 8192, 32, 8, 128, "bf16", 16),
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _lengths(case):
    """The lengths of a case's sequences; the longest one has ``high`` tokens."""
    rng = random.Random(case["salt"] * 7919 + case["batch"])
    lengths = [_log_uniform(rng, case["low"], case["high"]) for _ in range(case["batch"])]
    lengths[0] = case["high"]
    return lengths


def _fits(case):
    lengths = _lengths(case)
    tokens, longest = sum(lengths), case["high"]
    if case["op"] == "packed":
        wide = max(case["headdim"], 64) / 128
        cost = case["batch"] * case["heads"] * longest**2 * wide
        return (case["batch"] * case["heads"] * longest**2 <= _MOST_SCORES and cost <= _MOST_SCORES
                and tokens <= _MOST_TOKENS and tokens * case["heads"] * case["headdim"] <= _MOST_TOKENS * 16 * 128)
    width = case["kv_heads"] * case["headdim"]
    if case["batch"] * longest * width > _MOST_CACHE:
        return False
    if case["op"] == "append":
        fresh = tokens if case["fresh"] == "prompt" else case["batch"]
        return fresh * width <= _MOST_FRESH and fresh * case["heads"] * case["headdim"] <= 4 * _MOST_FRESH
    return True


def draw(rng):
    while True:
        op = rng.choice(["packed", "packed", "append", "decode"])
        kv_heads = rng.choice([1, 2, 2, 3, 4, 4, 8, 8])
        group = rng.choice([1, 1, 2, 3, 4, 4, 5, 8, 8, 16])
        dtype = rng.choice(["fp16", "bf16", "bf16"])
        headdim = rng.choice([32, 40, 64, 64, 72, 80, 96, 128, 128, 128])
        salt = rng.randrange(1, 1000000)
        if op == "packed":
            high = _log_uniform(rng, 16, 8192)
            low = rng.choice([high, max(1, high // 8), max(1, high // 2)])
            case = _packed("", rng.choice(["forward", "train", "train"]), _log_uniform(rng, 1, 64), low, high,
                           kv_heads * group, kv_heads, headdim, dtype, rng.choice(["dense", "dense", "fused"]),
                           rng.choice([0, 0, rng.randrange(1, 300)]), salt)
        elif op == "append":
            fresh = rng.choice(["token", "prompt"])
            high = _log_uniform(rng, 16, 8192)
            rotary = rng.choice([headdim // 16 * 16, headdim // 16 * 16, headdim // 32 * 16, 0])
            case = _append("", fresh, _log_uniform(rng, 1, 512 if fresh == "token" else 64), max(1, high // 16), high,
                           kv_heads * group, kv_heads, headdim, dtype, rng.choice([8, 16, 16, 24, 32, 64, 128]),
                           rotary, rotary > 0 and rng.random() < 0.3, salt)
        else:
            high = _log_uniform(rng, 16, 131072)
            headdim = rng.choice([headdim, headdim, 192, 256])
            case = _decode("", _log_uniform(rng, 1, 256), max(1, high // 16), high, kv_heads * group, kv_heads,
                           headdim, dtype, rng.choice([1, 8, 16, 16, 24, 32, 64, 128]), salt)
        if _fits(case):
            del case["name"]
            return case


def _in_order(case, seed):
    lengths = _lengths(case)
    random.Random(seed).shuffle(lengths)
    return lengths


def _tables(positions, rotary, device):
    """Cosines and sines of position x 10000^(-2 i / rotary), formed in 64 bits and kept in 32."""
    i = torch.arange(rotary // 2, device=device, dtype=torch.float64)
    angle = torch.arange(positions, device=device, dtype=torch.float64)[:, None] * 10000.0 ** (-2 * i / rotary)
    return angle.cos().float(), angle.sin().float()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, heads, kv_heads, d = _DTYPES[case["dtype"]], case["heads"], case["kv_heads"], case["headdim"]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g, dtype=dtype)

    def whole(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    lengths = _in_order(case, seed)
    starts = [0]
    for n in lengths:
        starts.append(starts[-1] + n)
    if case["op"] == "packed":
        rows = starts[-1] + case["behind"]
        state = {"case": case, "cu_seqlens": whole(starts), "longest": case["high"]}
        if case["layout"] == "fused":
            state["leaves"] = [normal(rows, heads + 2 * kv_heads, d)]
        else:
            state["leaves"] = [normal(rows, heads, d), normal(rows, kv_heads, d), normal(rows, kv_heads, d)]
        if case["direction"] == "train":
            for t in state["leaves"]:
                t.requires_grad_(True)
            state["d_output"] = normal(rows, heads, d)
        return state
    # a cache with a few pages to spare, handed out in no order
    page = case["page"]
    used = [-(-n // page) for n in lengths]
    pages = sum(used) + 3
    free = torch.randperm(pages, device="cuda", generator=g, dtype=torch.int32)
    table = torch.zeros(case["batch"], max(used), device="cuda", dtype=torch.int32)
    slot = torch.arange(max(used), device="cuda")
    inside = slot < whole(used)[:, None]
    table[inside] = free[: sum(used)]
    state = {"case": case, "block_table": table, "lengths": whole(lengths),
             "k_cache": normal(pages, page, kv_heads, d), "v_cache": normal(pages, page, kv_heads, d)}
    if case["op"] == "decode":
        state["q"] = normal(case["batch"], heads, d)
        return state
    prompt = case["fresh"] == "prompt"
    tokens = starts[-1] if prompt else case["batch"]
    state["cu_seqlens"] = whole(starts) if prompt else None
    state["q"], state["k"], state["v"] = (normal(tokens, h, d) for h in (heads, kv_heads, kv_heads))
    state["cos"], state["sin"] = _tables(case["high"], case["rotary"], "cuda") if case["rotary"] else (None, None)
    return state


# ------------------------------------------------------------------------------------------------ plain forms
def _projections(state):
    case, leaves = state["case"], state["leaves"]
    return leaves if case["layout"] == "dense" else leaves[0].split([case["heads"], case["kv_heads"], case["kv_heads"]], 1)


def _plain_packed(q, k, v, cu_seqlens, longest):
    rows, heads, d = q.shape
    kv_heads = k.shape[1]
    start, length = cu_seqlens[:-1].long(), (cu_seqlens[1:] - cu_seqlens[:-1]).long()
    at = torch.arange(longest, device=q.device)
    where = (start[:, None] + at).clamp_(max=rows - 1)  # rows of the padded batch
    qp, kp, vp = (t.float()[where].transpose(1, 2) for t in (q, k, v))  # [batch, heads, longest, d]
    batch = qp.shape[0]
    qp = qp.reshape(batch, kv_heads, -1, d)  # the query heads of a key head, one behind the other
    scores = (qp @ kp.transpose(2, 3)).view(batch, heads, longest, longest) * d**-0.5
    seen = (at[None, :] <= at[:, None]) & (at < length[:, None])[:, None, None, :]
    scores = scores.masked_fill(~seen, -math.inf)
    weights = (scores - scores.detach().amax(3, keepdim=True)).exp()
    weights = weights / weights.sum(3, keepdim=True)
    out = (weights.view(batch, kv_heads, -1, longest) @ vp).view(batch, heads, longest, d)
    row = torch.arange(rows, device=q.device)
    sequence = torch.searchsorted(cu_seqlens, row.to(torch.int32), right=True) - 1
    inside = sequence < batch
    sequence = sequence.clamp(max=batch - 1)
    out = out[sequence, :, (row - start[sequence]).clamp(max=longest - 1)]
    return torch.where(inside[:, None, None], out, 0.0).to(q.dtype)


def _plain_rotated(x, cos, sin, interleaved):
    half = cos.shape[1]
    x = x.float()
    cos, sin = cos[:, None], sin[:, None]
    head, rest = x[..., : 2 * half], x[..., 2 * half :]
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
        return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), rest], -1)
    a, b = head[..., :half], head[..., half:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)


def _plain_append(state):
    case, table, lengths = state["case"], state["block_table"], state["lengths"].long()
    q, k, v, cu_seqlens = state["q"], state["k"], state["v"], state["cu_seqlens"]
    row = torch.arange(k.shape[0], device=k.device)
    if cu_seqlens is None:
        sequence, position = row, lengths - 1
    else:
        sequence = torch.searchsorted(cu_seqlens, row.to(torch.int32), right=True) - 1
        position = lengths[sequence] - cu_seqlens[sequence + 1] + row
    if state["cos"] is not None:
        cos, sin = state["cos"][position], state["sin"][position]
        q, k = (_plain_rotated(t, cos, sin, case["interleaved"]).to(t.dtype) for t in (q, k))
    page = table[sequence, position // case["page"]].long()
    state["k_cache"][page, position % case["page"]] = k
    state["v_cache"][page, position % case["page"]] = v
    return (q, k) if case["fresh"] == "prompt" else (q,)


def _plain_decode(q, k_cache, v_cache, table, lengths):
    batch, heads, d = q.shape
    kv_heads = k_cache.shape[2]
    k, v = (t[table.long()].flatten(1, 2).float() for t in (k_cache, v_cache))  # [batch, keys, kv_heads, d]
    scores = q.float().view(batch, kv_heads, -1, d) @ k.permute(0, 2, 3, 1) * d**-0.5
    seen = torch.arange(k.shape[1], device=q.device) < lengths[:, None]
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    weights = (scores - scores.amax(3, keepdim=True)).exp()
    weights = weights / weights.sum(3, keepdim=True)
    return (weights @ v.transpose(1, 2)).view(batch, heads, d).to(q.dtype)


def run(state):
    case = state["case"]
    if own:
        from flash_attention_triton_b200 import append_kv_cache, flash_attention_decode, flash_attention_packed
    if case["op"] == "decode":
        with torch.no_grad():
            arguments = [state[key] for key in ("q", "k_cache", "v_cache", "block_table", "lengths")]
            return flash_attention_decode(*arguments) if own else _plain_decode(*arguments)
    if case["op"] == "append":
        with torch.no_grad():
            if own:
                prompt = case["fresh"] == "prompt"
                q, k = append_kv_cache(
                    state["k"], state["v"], state["k_cache"], state["v_cache"], state["block_table"], state["lengths"],
                    cu_seqlens=state["cu_seqlens"], q=state["q"], cos=state["cos"], sin=state["sin"],
                    interleaved=case["interleaved"], return_k=prompt)
                rotated = (q, k) if prompt else (q,)
            else:
                rotated = _plain_append(state)
            return [*rotated, state["k_cache"], state["v_cache"]]
    with torch.set_grad_enabled(case["direction"] == "train"):
        q, k, v = _projections(state)
        if own:
            out = flash_attention_packed(q, k, v, state["cu_seqlens"])
        else:
            out = _plain_packed(q, k, v, state["cu_seqlens"], state["longest"])
    if case["direction"] == "forward":
        return out
    return [out.detach(), *torch.autograd.grad(out, state["leaves"], state["d_output"])]


# ------------------------------------------------------------------------------------------------ in 64 bits
def _exact_packed(state):
    """Attention and its gradients, one sequence and head after the other, by the formulas."""
    case = state["case"]
    heads, kv_heads, d = case["heads"], case["kv_heads"], case["headdim"]
    q, k, v = (t.detach().double() for t in _projections(state))
    train = case["direction"] == "train"
    do = state["d_output"].double() if train else None
    out, dq, dk, dv = (torch.zeros_like(t) for t in (q, q, k, v))
    bounds = state["cu_seqlens"].tolist()
    for a, b in zip(bounds, bounds[1:]):
        behind = torch.ones(b - a, b - a, device=q.device, dtype=torch.bool).triu_(1)
        for h in range(heads):
            j = h * kv_heads // heads
            s = q[a:b, h] @ k[a:b, j].T / math.sqrt(d)
            s[behind] = -math.inf
            p = torch.softmax(s, 1)
            del s
            out[a:b, h] = p @ v[a:b, j]
            if train:
                dv[a:b, j] += p.T @ do[a:b, h]
                ds = do[a:b, h] @ v[a:b, j].T
                ds -= (do[a:b, h] * out[a:b, h]).sum(1, keepdim=True)
                ds *= p
                ds /= math.sqrt(d)
                dq[a:b, h] = ds @ k[a:b, j]
                dk[a:b, j] += ds.T @ q[a:b, h]
    if not train:
        return out
    return [out, torch.cat([dq, dk, dv], 1)] if case["layout"] == "fused" else [out, dq, dk, dv]


def _exact_append(state):
    """The cache entry by entry: each new token's keys and values at its place, the others as they were."""
    case = state["case"]
    q, k, v, k_cache, v_cache = (state[key].double() for key in ("q", "k", "v", "k_cache", "v_cache"))
    lengths, table, page = state["lengths"].tolist(), state["block_table"].tolist(), case["page"]
    if case["fresh"] == "prompt":
        bounds = state["cu_seqlens"].tolist()
        placed = [(n - (b - a) + i, s) for s, (a, b, n) in enumerate(zip(bounds, bounds[1:], lengths)) for i in range(b - a)]
    else:
        placed = [(n - 1, s) for s, n in enumerate(lengths)]
    position = torch.tensor([p for p, _ in placed], device=q.device)
    if case["rotary"]:
        c, s = (t.double()[position][:, None].to(torch.complex128) for t in (state["cos"], state["sin"]))
        turn, r = c + 1j * s, case["rotary"]
        for x in (q, k):
            first, second = (x[..., 0:r:2], x[..., 1:r:2]) if case["interleaved"] else (x[..., : r // 2], x[..., r // 2 : r])
            turned = torch.complex(first, second) * turn
            first.copy_(turned.real)
            second.copy_(turned.imag)
    entry = torch.tensor([table[s][p // page] * page + p % page for p, s in placed], device=q.device)
    k_cache.flatten(0, 1).index_copy_(0, entry, k)
    v_cache.flatten(0, 1).index_copy_(0, entry, v)
    return [q, k, k_cache, v_cache] if case["fresh"] == "prompt" else [q, k_cache, v_cache]


def _exact_decode(state):
    """One sequence after the other over the keys and values of its own pages."""
    case = state["case"]
    q, d = state["q"].double(), case["headdim"]
    out = torch.empty_like(q)
    group = case["heads"] // case["kv_heads"]
    for s, n in enumerate(state["lengths"].tolist()):
        pages = state["block_table"][s, : -(-n // case["page"])].long()
        for j in range(case["kv_heads"]):
            k, v = (state[key][pages, :, j].reshape(-1, d)[:n].double() for key in ("k_cache", "v_cache"))
            p = torch.softmax(q[s, j * group : (j + 1) * group] @ k.T / math.sqrt(d), 1)
            out[s, j * group : (j + 1) * group] = p @ v
    return out


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return {"packed": _exact_packed, "append": _exact_append, "decode": _exact_decode}[case["op"]](state)


def work(case):
    """packed: q, k, v (and dO) read, O (and dq, dk, dv) written once; two products of 2 d operations per pair that the
    mask keeps forward, five backward.  append: the new tokens read and written (q and, for prompts, k once more), their
    rows of the rotation tables.  decode: the keys and values of every sequence's length, and q and O."""
    lengths = _lengths(case)
    heads, kv_heads, d, tokens = case["heads"], case["kv_heads"], case["headdim"], sum(lengths)
    if case["op"] == "packed":
        pairs = sum(n * (n + 1) // 2 for n in lengths)
        train = case["direction"] == "train"
        sides = 2 if train else 1
        return {"bytes": 2 * d * tokens * ((2 * sides) * heads + 2 * sides * kv_heads),
                "flops": (14 if train else 4) * heads * pairs * d}
    if case["op"] == "append":
        prompt = case["fresh"] == "prompt"
        fresh = tokens if prompt else case["batch"]
        tables = 4 * (case["high"] if prompt else case["batch"]) * case["rotary"]
        return {"bytes": 2 * d * fresh * (2 * heads + (5 if prompt else 4) * kv_heads) + tables + 4 * fresh,
                "flops": 3 * fresh * (heads + kv_heads) * case["rotary"]}
    return {"bytes": 2 * d * (2 * tokens * kv_heads + 2 * case["batch"] * heads), "flops": 4 * tokens * heads * d}
