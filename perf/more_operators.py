"""The attention half of a block around its projections, as cases that can be timed: positions, the paged cache and the attention over it.

A case is a dict of plain values; its ``kind`` names the operator:

* ``rotary``  ``ops.rotary``: queries and keys are turned by their positions, in both layouts of the pairs, the whole head or a part of
              it, with the gradients of a training step (``train``);
* ``append``  ``ops.cache_append``: the new tokens' keys (rotated on the way) and values are written to their sequences' pages, their
              queries rotated in the same call;
* ``attend``  ``ops.cached_attention``: the new tokens attend to a prefix that all sequences share, and to their own sequence's pages.

``own`` false: the operators in elementary torch operations, in 32 bits (angles in 64); true: the framework's kernels.

The cache keeps a head's keys and values of a page in tiles of four 16-byte groups of keys; E is the number of elements in 16 bytes:

* keys    ``[place / 4E][feature / 4E][half][group of features][place / E][place % 4][E features]``, ``half`` = ``place % E / 4``;
* values  ``[place / 4E][feature / 16][place / E][feature % 16][E places]``.
"""

import math
import random

import torch

own = False

_DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}


def _rotary_case(name, tokens, heads, kv_heads, dim, rotary_dim, dtype, interleaved=False, far=0, scaled=False, train=False):
    return dict(name=name, kind="rotary", tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, rotary_dim=rotary_dim, dtype=dtype,
                interleaved=interleaved, far=far, scaled=scaled, train=train)


def _append_case(name, sequences, new, context, heads, kv_heads, dim, rotary_dim, page, dtype, interleaved=False, ragged=False, prefix=0):
    return dict(name=name, kind="append", sequences=sequences, new=new, context=context, heads=heads, kv_heads=kv_heads, dim=dim,
                rotary_dim=rotary_dim, page=page, dtype=dtype, interleaved=interleaved, ragged=ragged, prefix=prefix)


def _attend_case(name, sequences, new, context, heads, kv_heads, dim, page, dtype, ragged=False, prefix=0):
    return dict(name=name, kind="attend", sequences=sequences, new=new, context=context, heads=heads, kv_heads=kv_heads, dim=dim,
                page=page, dtype=dtype, ragged=ragged, prefix=prefix)


def listed():
    return [
        # One decoded token of the 2B-parameter stack, outside a cache: the smallest call, launch and host latency.
        _rotary_case("rotary_token", 1, 20, 20, 128, 128, "bf16", far=700),
        # A long document's tokens with far, scaled positions, neighbouring pairs and a part of an odd head; training.
        _rotary_case("rotary_ragged", 777, 12, 4, 80, 32, "fp16", interleaved=True, far=500000, scaled=True, train=True),
        # A training step's share of one block of the 2B-parameter stack over 8 x 512 tokens.
        _rotary_case("rotary_train", 4096, 20, 20, 128, 128, "bf16", train=True),
        # One step of a batch of 64 conversations with shared key heads.
        _append_case("append_batch", 64, 1, 500, 32, 8, 128, 128, 64, "bf16"),
        # Chunks of unlike lengths (some sequences get nothing) behind a shared prefix, an odd head dimension, half precision.
        _append_case("append_ragged", 37, 200, 900, 10, 2, 80, 32, 32, "fp16", interleaved=True, ragged=True, prefix=1000),
        # The prompts of the 2B-parameter stack, 8 x 512 tokens, into empty pages.
        _append_case("append_prompt", 8, 512, 512, 20, 20, 128, 128, 64, "bf16"),
        # One token of one short conversation through the 2B-parameter stack: latency.
        _attend_case("attend_token", 1, 1, 500, 20, 20, 128, 64, "bf16"),
        # A few drafted tokens a sequence (some have none) behind a shared prefix, an odd head dimension, half precision.
        _attend_case("attend_ragged", 37, 7, 900, 10, 2, 80, 32, "fp16", ragged=True, prefix=1000),
        # One token of one very long conversation: the keys of one sequence fill the chip.
        _attend_case("attend_long", 1, 1, 100000, 32, 8, 128, 64, "bf16"),
        # One step of a batch of 64 conversations of up to four thousand tokens.
        _attend_case("attend_batch", 64, 1, 4096, 32, 8, 128, 64, "bf16"),
        # One step of a batch of 128 short answers to one long document.
        _attend_case("attend_prefix", 128, 1, 512, 32, 8, 128, 64, "bf16", prefix=16384),
        # Prompts in chunks: 4 x 512 new tokens on what their sequences hold already.
        _attend_case("attend_chunk", 4, 512, 4096, 32, 8, 128, 64, "bf16"),
    ]


# ---- draws -----------------------------------------------------------------------------------------------------------

_MAX_ROTARY = 4096 * 40 * 128            # elements: rotary_train's
_MAX_APPEND = 8 * 512 * 60 * 128         # elements moved: append_prompt's
_MAX_CACHE = 64 * 4096 * 8 * 128         # keys' elements: attend_batch's


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _head(rng):
    return rng.choice((64, 80, 96, 128, 128, 128, 192, 256, rng.randrange(16, 257)))


def _heads(rng):
    kv = rng.choice((1, 2, 4, 8, 8, 20, rng.randrange(1, 17)))
    return kv * rng.choice((1, 1, 2, 4, 4, 5, 8)), kv


def draw(rng):
    while True:
        kind = rng.choice(("rotary", "append", "attend", "attend"))
        dtype, dim, (heads, kv) = rng.choice(("bf16", "bf16", "fp16", "fp32")), _head(rng), _heads(rng)
        part = rng.choice((dim // 2 * 2, dim // 2 * 2, dim // 4 * 2))
        if kind == "rotary":
            case = dict(kind=kind, tokens=rng.choice((_log_uniform(rng, 1, 64), _log_uniform(rng, 64, 32768))), heads=heads, kv_heads=kv,
                        dim=dim, rotary_dim=part, dtype=dtype, interleaved=rng.random() < 0.4,
                        far=rng.choice((0, 0, _log_uniform(rng, 1000, 1000000))), scaled=rng.random() < 0.3, train=rng.random() < 0.5)
            if case["tokens"] * (heads + kv) * dim <= _MAX_ROTARY:
                return case
            continue
        new = rng.choice((1, 1, 1, _log_uniform(rng, 2, 16), _log_uniform(rng, 16, 2048)))
        case = dict(kind=kind, sequences=_log_uniform(rng, 1, 256), new=new, context=max(new, _log_uniform(rng, 16, 131072)), heads=heads,
                    kv_heads=kv, dim=dim, page=rng.choice((32, 64, 64, 128, 256)), dtype=dtype, ragged=rng.random() < 0.5,
                    prefix=rng.choice((0, 0, _log_uniform(rng, 1, 32768))))
        held, tokens = case["sequences"] * case["context"] * kv * dim, case["sequences"] * new
        if kind == "append":
            case.update(rotary_dim=part, interleaved=rng.random() < 0.4)
            if held <= _MAX_CACHE // 4 and tokens * (heads + 2 * kv) * dim <= _MAX_APPEND:
                return case
        elif (held + case["prefix"] * kv * dim) * _SIZE[dtype] <= 2 * _MAX_CACHE:
            pairs = tokens * heads * (case["context"] + case["prefix"])  # (the plain form keeps as many weights in 32 bits)
            if pairs <= 512 * 4 * 32 * 4096 // (8 if dtype == "fp32" else 1) and pairs * dim <= 512 * 4 * 32 * 4096 * 128 // (8 if dtype == "fp32" else 1):
                return case


def _batch(case):
    """Each sequence's new tokens and its length with them: of the case alone, since the work goes by them."""
    rng = random.Random(f"{case['sequences']} {case['new']} {case['context']} {case['ragged']}")
    new = [rng.randint(0, case["new"]) if case["ragged"] else case["new"] for _ in range(case["sequences"])]
    if case["ragged"] and not any(new):
        new[0] = case["new"]
    full = case["new"] == case["context"] or case["sequences"] == 1
    held = [case["context"] if full else rng.randint(max(case["new"], case["context"] // 4), case["context"]) for _ in new]
    return new, held


# ---- what a program holds before the call ----------------------------------------------------------------------------

def _normal(g, shape, std, dtype=torch.float32):
    return torch.randn(shape, generator=g, device=g.device).mul_(std).to(dtype)


def _frequencies(rotary_dim, scaled, device):
    """1 / 10000^(2i / rotary_dim), in 64 bits; scaled: long waves four times as long, with a ramp up to there."""
    f = 10000.0 ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim)
    if scaled:
        keep = ((8192 * f / (2 * math.pi) - 1) / 31).clamp(0, 1)
        f = f * keep + f / 4 * (1 - keep)
    return f


def _tiled(k, v):
    """Pages ``[pages, heads, places, features]`` of keys and values in the cache's order."""
    (n, h, p, d), e = k.shape, 16 // k.element_size()
    tiles = p // (4 * e)
    # place = (tile, p/E, half, p%4), feature = (chunk, group, e)
    kt = k.view(n, h, tiles, 4, e // 4, 4, d // (4 * e), 4, e).permute(0, 1, 2, 6, 4, 7, 3, 5, 8)
    vt = v.view(n, h, tiles, 4, e, d // 16, 16).permute(0, 1, 2, 5, 3, 6, 4)
    return kt.reshape(n, h, p, d), vt.reshape(n, h, p, d)


def _pages(total, page):
    return (total + page - 1) // page


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 6151 + 17)
    dev, dt, dim, heads, kv = g.device, _DTYPES[case["dtype"]], case["dim"], case["heads"], case["kv_heads"]
    state = dict(kind=case["kind"])
    if case["kind"] == "rotary":
        t = case["tokens"]
        state.update(q=_normal(g, (t, heads, dim), 1.0, dt), k=_normal(g, (t, kv, dim), 1.0, dt), train=case["train"],
                     positions=torch.arange(t, device=dev) + case["far"], interleaved=case["interleaved"],
                     inv_freq=_frequencies(case["rotary_dim"], case["scaled"], dev),
                     amplitude=0.1 * math.log(4.0) + 1.0 if case["scaled"] else 1.0)
        if case["train"]:
            state.update(dq=_normal(g, (t, heads, dim), 0.01, dt), dk=_normal(g, (t, kv, dim), 0.01, dt))
            state["q"].requires_grad_()
            state["k"].requires_grad_()
        return state
    page, unit = case["page"], 64 // _SIZE[case["dtype"]]
    new, held = _batch(case)
    padded, tokens = (dim + unit - 1) // unit * unit, sum(new)
    width, shared = _pages(case["context"], page), _pages(case["prefix"], page)
    pages = sum(_pages(n, page) for n in held) + shared + 3
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    state["prefix_table"], state["prefix_length"] = (order[:shared], case["prefix"]) if shared else (None, 0)
    table, at = torch.full((len(held), width), -1, dtype=torch.int32), shared
    order_cpu = order.cpu()
    for i, n in enumerate(held):
        table[i, :_pages(n, page)] = order_cpu[at:at + _pages(n, page)]
        at += _pages(n, page)
    kc, vc = (_normal(g, (pages, kv, page, padded), 1.0, dt) for _ in range(2))
    kc[..., dim:], vc[..., dim:] = 0, 0
    state["k_cache"], state["v_cache"] = _tiled(kc, vc)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    ragged = case["ragged"] or case["new"] > 1
    state.update(block_table=table.to(dev), lengths=torch.tensor(held, dtype=torch.int32, device=dev),
                 q_starts=torch.tensor(starts, dtype=torch.int32, device=dev) if ragged else None, most=max(new), dim=dim,
                 q=_normal(g, (tokens, heads, dim), 1.5, dt))
    if case["kind"] == "append":
        state.update(k=_normal(g, (tokens, kv, dim), 1.0, dt), v=_normal(g, (tokens, kv, dim), 1.0, dt), interleaved=case["interleaved"],
                     inv_freq=_frequencies(case["rotary_dim"], False, dev))
    return state


# ---- one pass --------------------------------------------------------------------------------------------------------

def run(state):
    if own:
        return {"rotary": _rotary_own, "append": _append_own, "attend": _attend_own}[state["kind"]](state)
    with torch.no_grad():
        return {"rotary": _rotary_plain, "append": _append_plain, "attend": _attend_plain}[state["kind"]](state)


def _rotary_own(st):
    from bittorch_amd import ops

    q, k = ops.rotary(st["q"], st["k"], st["positions"], st["inv_freq"], interleaved=st["interleaved"], amplitude=st["amplitude"])
    if not st["train"]:
        return dict(q=q, k=k)
    dq, dk = torch.autograd.grad((q, k), (st["q"], st["k"]), (st["dq"], st["dk"]))
    return dict(q=q.detach(), k=k.detach(), dq=dq, dk=dk)


def _append_own(st):
    from bittorch_amd import ops

    q = ops.cache_append(st["k"], st["v"], st["k_cache"], st["v_cache"], st["block_table"], st["lengths"], st["q_starts"], q=st["q"],
                         inv_freq=st["inv_freq"], interleaved=st["interleaved"], first_position=st["prefix_length"])
    return dict(q=q, k_cache=st["k_cache"], v_cache=st["v_cache"])


def _attend_own(st):
    from bittorch_amd import ops

    out, lse = ops.cached_attention(st["q"], st["k_cache"], st["v_cache"], st["block_table"], st["lengths"], st["q_starts"],
                                    prefix_table=st["prefix_table"], prefix_length=st["prefix_length"], return_lse=True)
    return dict(out=out, lse=lse)


def _turned(x, cos, sin, interleaved):
    """x with its pairs turned, in 32 bits; the features behind them as they are."""
    n, x = 2 * cos.shape[-1], x.float()
    part, rest = x[..., :n], x[..., n:]
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
        part = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = part[..., :n // 2], part[..., n // 2:]
        part = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((part, rest), -1)


def _angles(positions, inv_freq, amplitude=1.0):
    angle = positions.double()[:, None] * inv_freq
    return ((f(angle) * amplitude).float()[:, None, :] for f in (torch.cos, torch.sin))


def _rotary_plain(st):
    cos, sin = _angles(st["positions"], st["inv_freq"], st["amplitude"])
    out = {n: _turned(st[n], cos, sin, st["interleaved"]).to(st[n].dtype) for n in ("q", "k")}
    if st["train"]:
        out.update({n: _turned(st[n], cos, -sin, st["interleaved"]).to(st[n].dtype) for n in ("dq", "dk")})
    return out


def _owners(st):
    """Of each new token: its sequence, and its place there."""
    lengths, starts = st["lengths"].long(), st["q_starts"]
    if starts is None:
        return torch.arange(len(lengths), device=lengths.device), lengths - 1
    token = torch.arange(st["q"].shape[0], device=lengths.device)
    owner = torch.searchsorted(starts[1:].long(), token, right=True)
    return owner, lengths[owner] - starts[1:].long()[owner] + token


def _append_plain(st):
    owner, place = _owners(st)
    cos, sin = _angles(place + st["prefix_length"], st["inv_freq"])
    k, q = (_turned(st[n], cos, sin, st["interleaved"]).to(st[n].dtype) for n in ("k", "q"))
    (_, kv, page, padded), dim, e = st["k_cache"].shape, st["dim"], 16 // k.element_size()
    d, head = torch.arange(dim, device=k.device), torch.arange(kv, device=k.device)[None, :, None]
    at, r = place % page, place % (4 * e)
    block = (st["block_table"][owner, place // page].long()[:, None, None] * kv + head) * page * padded
    tile = (at // (4 * e) * 4 * e * padded)[:, None, None]
    col = lambda t: t[:, None, None]  # noqa: E731
    k_at = ((((d // (4 * e)) * (e // 4) + col(r % e // 4)) * 4 + d % (4 * e) // e) * 16 + col(r // e * 4 + r % 4)) * e + d % e
    v_at = ((d // 16 * 4 + col(r // e)) * 16 + d % 16) * e + col(r % e)
    st["k_cache"].view(-1)[block + tile + k_at] = k
    st["v_cache"].view(-1)[block + tile + v_at] = st["v"]
    return dict(q=q, k_cache=st["k_cache"], v_cache=st["v_cache"])


def _held(k_cache, v_cache, table, dim):
    """Keys and values of the pages of a table ``[..., width]`` in 32 bits: ``[..., heads, width * page, dim]``."""
    (_, h, p, d), e = k_cache.shape, 16 // k_cache.element_size()
    index = table.long().clamp(min=0)
    lead, width = index.shape[:-1], index.shape[-1]
    k = k_cache[index].float().view(-1, width, h, p // (4 * e), d // (4 * e), e // 4, 4, 4, 4, e)
    k = k.permute(0, 2, 1, 3, 7, 5, 8, 4, 6, 9).reshape(*lead, h, width * p, d)
    v = v_cache[index].float().view(-1, width, h, p // (4 * e), d // 16, 4, 16, e)
    v = v.permute(0, 2, 1, 3, 5, 7, 4, 6).reshape(*lead, h, width * p, d)
    return k[..., :dim], v[..., :dim]


def _attend_plain(st):
    q, lengths, kv, dim = st["q"], st["lengths"].long(), st["k_cache"].shape[1], st["dim"]
    (tokens, heads, _), n_seq, most = q.shape, len(lengths), st["most"]
    starts = torch.arange(n_seq + 1, device=q.device) if st["q_starts"] is None else st["q_starts"].long()
    new = starts[1:] - starts[:-1]
    # the queries by sequence, padded to the most that one has: [sequence, key head, head of the group and token, dim]
    step = torch.arange(most, device=q.device)
    row = torch.where(step < new[:, None], starts[:-1, None] + step, tokens)
    rows = torch.cat((q.float() / math.sqrt(dim), q.new_zeros(1, heads, dim, dtype=torch.float32)))[row]
    rows = rows.view(n_seq, most, kv, heads // kv, dim).permute(0, 2, 3, 1, 4).reshape(n_seq, kv, -1, dim)
    k, v = _held(st["k_cache"], st["v_cache"], st["block_table"], dim)
    logits = rows @ k.transpose(-1, -2)
    seen = torch.arange(k.shape[-2], device=q.device) <= (lengths - new)[:, None, None] + step[:, None]      # [sequence, token, key]
    logits = logits.view(n_seq, kv, -1, most, k.shape[-2]).masked_fill_(~seen[:, None, None], -math.inf).view(n_seq, kv, -1, k.shape[-2])
    top = logits.amax(-1, keepdim=True)
    if st["prefix_length"]:
        pk, pv = _held(st["k_cache"], st["v_cache"], st["prefix_table"], dim)
        pk, pv = pk[:, :st["prefix_length"]], pv[:, :st["prefix_length"]]
        flat = rows.transpose(0, 1).reshape(kv, -1, dim)                                                     # every sequence's, by key head
        shared = flat @ pk.transpose(-1, -2)
        back = lambda t: t.view(kv, n_seq, -1, t.shape[-1]).transpose(0, 1)  # noqa: E731
        top = torch.maximum(top, back(shared.amax(-1, keepdim=True)))
        shared = torch.exp_(shared - top.transpose(0, 1).reshape(kv, -1, 1))
        total, out = back(shared.sum(-1, keepdim=True)), back(shared @ pv)
    else:
        total, out = 0.0, 0.0
    weights = torch.exp_(logits.sub_(top))
    total = total + weights.sum(-1, keepdim=True)
    out, lse = (out + weights @ v) / total, top + torch.log(total)
    by_token = lambda t: t.view(n_seq, kv, heads // kv, most, -1).permute(0, 3, 1, 2, 4).reshape(n_seq * most, heads, -1)  # noqa: E731
    result, sums = q.new_empty(tokens + 1, heads, dim), torch.empty(tokens + 1, heads, 1, device=q.device)
    result[row.reshape(-1)], sums[row.reshape(-1)] = by_token(out).to(q.dtype), by_token(lse)
    return dict(out=result[:tokens], lse=sums[:tokens, :, 0])


# ---- what a pass cannot do without -----------------------------------------------------------------------------------

def work(case):
    size, heads, kv, dim = _SIZE[case["dtype"]], case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "rotary":
        passes, n = (2 if case["train"] else 1), case["tokens"] * (heads + kv)
        return {"bytes": passes * 2 * size * n * dim + 8 * case["tokens"], "flops": passes * 3.0 * n * case["rotary_dim"]}
    new, held = _batch(case)
    tokens = sum(new)
    if case["kind"] == "append":
        return {"bytes": 2 * size * tokens * (heads + 2 * kv) * dim, "flops": 3.0 * tokens * (heads + kv) * case["rotary_dim"]}
    keys = sum(h for n, h in zip(new, held) if n) + case["prefix"]
    pairs = sum(n * (h - n) + n * (n + 1) // 2 for n, h in zip(new, held)) + tokens * case["prefix"]
    return {"bytes": 2 * size * (keys * kv + tokens * heads) * dim + 4 * tokens * heads, "flops": 4.0 * pairs * heads * dim}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------

def _exact_turn(x, positions, inv_freq, interleaved, amplitude, backward=False):
    """Complex multiplication by amplitude * exp(i * position * frequency)."""
    n = 2 * inv_freq.numel()
    x = x.detach().double()
    angle = torch.outer(positions.double(), inv_freq)
    unit = torch.polar(torch.full_like(angle, amplitude), -angle if backward else angle)[:, None]
    if interleaved:
        turned = torch.view_as_real(torch.view_as_complex(x[..., :n].reshape(*x.shape[:-1], n // 2, 2).contiguous()) * unit).reshape(*x.shape[:-1], n)
    else:
        z = torch.complex(x[..., :n // 2], x[..., n // 2:n]) * unit
        turned = torch.cat((z.real, z.imag), -1)
    return torch.cat((turned, x[..., n:]), -1)


def _exact_places(st, new, held, page):
    """Of every sequence: its table row and its places as (page, place in it)."""
    table = st["block_table"].cpu().tolist()
    for i, (n, h) in enumerate(zip(new, held)):
        places = torch.arange(h)
        yield n, h, torch.tensor(table[i], dtype=torch.long)[places // page], places % page


def exact(case, seed):
    st = prepare(case, seed)
    dim, kv, heads = case["dim"], case["kv_heads"], case["heads"]
    if case["kind"] == "rotary":
        args = st["positions"], st["inv_freq"], st["interleaved"], st["amplitude"]
        out = {n: _exact_turn(st[n], *args) for n in ("q", "k")}
        if case["train"]:
            out.update({n: _exact_turn(st[n], *args, backward=True) for n in ("dq", "dk")})
        return out
    new, held = _batch(case)
    page, e = case["page"], 16 // _SIZE[case["dtype"]]
    padded = st["k_cache"].shape[-1]

    def natural(kc, vc):
        n = kc.shape[0]
        k = kc.double().view(n, kv, page // (4 * e), padded // (4 * e), e // 4, 4, 4, 4, e)
        k = torch.einsum("nhtcugpqe->nhtpuqcge", k).reshape(n, kv, page, padded)
        v = torch.einsum("nhtbgde->nhtgebd", vc.double().view(n, kv, page // (4 * e), padded // 16, 4, 16, e)).reshape(n, kv, page, padded)
        return k, v

    if case["kind"] == "append":
        k, v = natural(st["k_cache"], st["v_cache"])
        position = torch.cat([torch.arange(h - n, h) for n, h in zip(new, held)]).to(k.device) + case["prefix"]
        turned = [_exact_turn(st[n], position, st["inv_freq"], st["interleaved"], 1.0) for n in ("q", "k")]
        at = [(p[h - n:], r[h - n:]) for n, h, p, r in _exact_places(st, new, held, page)]
        p, r = (torch.cat(t).to(k.device) for t in zip(*at))
        k[p, :, r, :dim], v[p, :, r, :dim] = turned[1], st["v"].double()
        k = torch.einsum("nhtpuqcge->nhtcugpqe", k.view(-1, kv, page // (4 * e), 4, e // 4, 4, padded // (4 * e), 4, e))
        v = torch.einsum("nhtgebd->nhtbgde", v.view(-1, kv, page // (4 * e), 4, e, padded // 16, 16))
        return dict(q=turned[0], k_cache=k.reshape(-1, kv, page, padded), v_cache=v.reshape(-1, kv, page, padded))
    q, out, lse, at = st["q"].double(), [], [], 0
    shared = None
    if case["prefix"]:
        k, v = natural(st["k_cache"][st["prefix_table"].long()], st["v_cache"][st["prefix_table"].long()])
        shared = [t.transpose(0, 1).reshape(kv, -1, padded)[:, :case["prefix"], :dim] for t in (k, v)]
    for n, h, p, r in _exact_places(st, new, held, page):
        if n == 0:
            continue
        k, v = natural(st["k_cache"][p[::page].to(q.device)], st["v_cache"][p[::page].to(q.device)])
        k, v = (t.transpose(0, 1).reshape(kv, -1, padded)[:, :h, :dim] for t in (k, v))
        mask = torch.ones(n, h, dtype=torch.bool, device=q.device).tril(h - n)
        if shared:
            k, v = torch.cat((shared[0], k), 1), torch.cat((shared[1], v), 1)
            mask = torch.cat((mask.new_ones(n, case["prefix"]), mask), 1)
        rows = q[at:at + n].transpose(0, 1).reshape(kv, heads // kv, n, dim)
        s = (rows.flatten(1, 2) @ k.mT / dim ** 0.5).view(kv, heads // kv, n, -1).masked_fill(~mask, -math.inf)
        lse.append(s.logsumexp(-1).flatten(0, 1).T)
        out.append((s.softmax(-1).flatten(1, 2) @ v).view(heads, n, dim).transpose(0, 1))
        at += n
    return dict(out=torch.cat(out), lse=torch.cat(lse))
