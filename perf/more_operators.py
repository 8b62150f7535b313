"""A stream's queries, keys and its cache in 8 bits, as cases that can be timed and compared.

A case is a dict of plain values.  ``listed()`` names the ones that are always looked at, ``draw(rng)`` makes more of the
same ranges, ``prepare`` builds what a program holds before the call, ``run`` makes one pass (the framework's kernels where
``own`` is true, elementary torch operations in 32 bits where it is not), ``exact`` is the same in 64 bits from the
definition, and ``work`` says what the pass cannot do without.

Five kinds of work, around the sliding-window attention of a stream (sinks + window rows of cache, a ring behind the sinks; the
token at position p is row p below the sinks, else row sinks + (p - sinks) % window):

* ``rope``    the heads of queries and keys are normed (root mean square over the head, weights) and rotated by their position, on the
              views of a fused projection: channel pairs (2i, 2i + 1) or (i, i + rotary / 2), the first ``rotary`` channels of the head,
* ``append``  new tokens' keys and values go into a cache of 8 bits, which is then read whole and in order (what the next chunk's
              attention takes),
* ``turn``    both: norm and rotation, queries out, keys and values into the cache of 8 bits, the cache read whole,
* ``read``    the rows of a cache in the order of their tokens: sinks, then the last ``window`` tokens,
* ``attend``  one token of each stream over a cache of 8 bits that holds it already.

In 8 bits a head's row x is whole numbers c = round(127 x / max|x|), ties to even, and a scale max|x| / 127 (the scales
of a row's key and value lie side by side).  Widths are those of the image and video models here (1152 and 2240 channels, heads of
32, 72 and 112) and generic ones (heads of 64 and 128); 1560 tokens are a latent frame of 480p, 4680 the three frames of a streamed chunk.
"""
import math

import torch

own = False
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6
BASE = 10000.0


def _rope(name, batch, tokens, heads, kv_heads, dim, rotary, *, pairs="near", first=0, scaled=1.0, dtype="bf16", ragged=False):
    return {"name": name, "kind": "rope", "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rotary": rotary,
            "pairs": pairs, "first": first, "scaled": scaled, "dtype": dtype, "ragged": ragged}


def _append(name, batch, tokens, kv_heads, dim, window, sinks, *, dtype="bf16"):
    return {"name": name, "kind": "append", "batch": batch, "tokens": tokens, "kv_heads": kv_heads, "dim": dim, "window": window, "sinks": sinks,
            "dtype": dtype}


def _turn(name, batch, tokens, heads, kv_heads, dim, rotary, window, sinks, *, pairs="near", dtype="bf16"):
    return {"name": name, "kind": "turn", "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rotary": rotary,
            "pairs": pairs, "scaled": 1.0, "window": window, "sinks": sinks, "dtype": dtype}


def _read(name, batch, kv_heads, dim, window, sinks, *, bits=8, dtype="bf16"):
    return {"name": name, "kind": "read", "batch": batch, "kv_heads": kv_heads, "dim": dim, "window": window, "sinks": sinks, "bits": bits,
            "dtype": dtype}


def _attend(name, batch, heads, kv_heads, dim, window, sinks, *, dtype="bf16"):
    return {"name": name, "kind": "attend", "batch": batch, "heads": heads, "kv_heads": kv_heads, "dim": dim, "window": window, "sinks": sinks,
            "dtype": dtype}


def listed():
    return [
        # one token of one stream at the width of the small image model: nothing but latency
        _rope("rope_token_b1", 1, 1, 16, 16, 72, 72),
        # the tokens of one large image in scan order
        _rope("rope_16384", 1, 16384, 20, 20, 112, 112),
        # prompts of unlike length that continue far into their streams: shared key heads, half of the head rotated, frequencies scaled down
        _rope("rope_far_ragged_fp16", 8, 2047, 32, 8, 128, 64, pairs="far", first=1500000, scaled=8.0, dtype="fp16", ragged=True),
        # three streamed frames of two streams behind the first frame, which stays, and six of the past; shared key heads, half precision
        _append("append_chunk_fp16", 2, 4680, 5, 112, 9360, 1560, dtype="fp16"),
        # the last tokens of a batch of long prompts go into short caches
        _append("append_prompts_b16", 16, 4096, 4, 128, 2048, 4),
        # a streamed chunk from its projection into the caches, and what the next chunk will look back at
        _turn("turn_chunk_b2", 2, 4680, 20, 20, 112, 112, 9360, 1560),
        # a token of each stream of a serving batch, short windows
        _turn("turn_token_b48", 48, 1, 35, 35, 64, 32, 256, 4, pairs="far"),
        # a short 16-bit cache in order: latency
        _read("read_b1_16bit", 1, 16, 72, 256, 4, bits=16),
        # the past of two streams in front of their next chunk
        _read("read_chunk_b2", 2, 20, 112, 9360, 1560),
        # one stream, one token over a short window
        _attend("attend_b1", 1, 16, 16, 72, 1024, 4),
        # a full serving batch over long windows with shared key heads
        _attend("attend_gqa_b64", 64, 32, 8, 128, 8192, 4),
        # one stream over a very long window: all the card for one token
        _attend("attend_long_b1_fp16", 1, 32, 8, 128, 131072, 64, dtype="fp16"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rope", "append", "turn", "read", "attend"])
    heads, dim = rng.choice([(36, 32), (70, 32), (35, 64), (16, 72), (12, 96), (20, 112), (16, 128), (32, 128)])
    kv_heads = heads // rng.choice([g for g in (1, 2, 4, 5, 7, 8) if heads % g == 0])
    dtype = rng.choice(["bf16", "fp16"])
    rotated = {"rotary": 8 * rng.randint(max(1, dim // 32), dim // 8), "pairs": rng.choice(["near", "far"])}
    if kind == "rope":
        tokens = _log_int(rng, 1, 16000)
        return {"kind": kind, "batch": _log_int(rng, 1, max(1, min(64, 16000 // tokens))), "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
                "dim": dim, **rotated, "first": rng.choice([0, _log_int(rng, 1, 4000000)]), "scaled": rng.choice([1.0, 4.0]), "dtype": dtype,
                "ragged": rng.random() < 0.5}
    if kind == "attend":
        rows = _log_int(rng, 16, 60000)
        return {"kind": kind, "batch": _log_int(rng, 1, max(1, min(96, 200000 // rows))), "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "window": rows, "sinks": rng.choice([0, 1, 4, 64]), "dtype": dtype}
    window, sinks = _log_int(rng, 16, 6000), rng.choice([0, 1, 4, 64, 390])
    batch = _log_int(rng, 1, max(1, min(48, 16000 // (window + sinks))))
    common = {"kind": kind, "batch": batch, "kv_heads": kv_heads, "dim": dim, "window": window, "sinks": sinks, "dtype": dtype}
    if kind == "read":
        return {**common, "bits": rng.choice([8, 16])}
    tokens = rng.choice([1, _log_int(rng, 2, 3 * 4000 // batch + 2)])
    if kind == "append":
        return {**common, "tokens": tokens}
    return {**common, "tokens": tokens, "heads": heads, **rotated, "scaled": 1.0}


def _spread(count, lo, hi):
    """`count` whole numbers from lo to hi, evenly spread, hi among them."""
    return [hi - (hi - lo) * i // max(1, count - 1) for i in range(count)]


def _lengths(case):
    n = case["tokens"]
    return _spread(case["batch"], n // 2, n) if case.get("ragged") else [n] * case["batch"]


def _positions(case):
    """Tokens that each stream has seen: from just as many as its cache holds (attend: half as many) to three times that."""
    if case["kind"] == "rope":
        return _spread(case["batch"], case["first"] // 2, case["first"])
    full = case["sinks"] + case["window"]
    return _spread(case["batch"], full // 2 if case["kind"] == "attend" else full, 3 * full) if case["batch"] > 1 else [2 * full + 7]


def _frequencies(case):
    """Radians a position of each pair; scaled: pairs that turn less than once in 4096 positions are slowed, more than 32 times left as they
    are, a blend by their number of turns between."""
    i = torch.arange(case["rotary"] // 2, dtype=torch.float64, device="cuda")
    f = BASE ** (-2.0 * i / case["rotary"])
    turns = 4096 * f / (2 * math.pi)
    keep = ((turns - 1) / 31).clamp(0, 1)
    return f * (keep + (1 - keep) / case["scaled"])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt, B, G, d = DTYPES[case["dtype"]], case["batch"], case["kv_heads"], case["dim"]
    order = torch.randperm(B, generator=gen, device="cuda").cpu()

    def rows(values):
        return torch.tensor(values)[order].to(device="cuda", dtype=torch.int32)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)

    st = {"case": case, "positions": rows(_positions(case))}
    kind, T, H = case["kind"], case.get("tokens", 1), case.get("heads", 0)
    if kind != "read":
        qkv = normal(B, T, (H + 2 * G) * d).to(dt)
        st["q"], st["k"], st["v"] = qkv.split([H * d, G * d, G * d], dim=2)
    if kind in ("rope", "turn"):
        st["q_weight"], st["k_weight"] = ((1 + 0.2 * normal(d)).to(dt) for _ in range(2))
        st["freqs"] = _frequencies(case)
        st["lengths"] = rows(_lengths(case)) if case.get("ragged") else None
    if kind == "rope":
        return st
    st["after"] = st["positions"] + T     # what the program's streams have seen once the tokens are in
    held = case["sinks"] + case["window"]
    if case.get("bits") == 16:
        st["cache"] = tuple(normal(B, held, G * d).to(dt) for _ in range(2))
        return st
    # rows of normal values as they lie in 8 bits: the largest of a head is 127, some 2.7 times the rest's deviation; heads of 8 bits
    # lie in a multiple of 16 bytes
    width = -(-d // 16) * 16
    codes = [normal(B, G, held, width).mul_(46).round_().clamp_(-127, 127).to(torch.int8) for _ in range(2)]
    scales = torch.exp(0.2 * normal(B, G, held, 2)).mul_(2.7 / 127)
    st["cache"] = (*codes, scales)
    st["scale"] = d ** -0.5
    return st


def _heads(t, dim):
    """[B, N, heads * dim] -> fp32 [B, N, heads, dim]"""
    return t.unflatten(2, (-1, dim)).float()


def _normed(x, weight):
    return x * torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + EPS) * weight.to(x.dtype)


def _rotated(x, angle, case):
    """x [B, N, heads, dim] by angle [B, N, rotary / 2], 64 bits."""
    r = case["rotary"]
    cos, sin = torch.cos(angle).to(x.dtype)[:, :, None], torch.sin(angle).to(x.dtype)[:, :, None]
    if case["pairs"] == "near":
        a, b = x[..., 0:r:2], x[..., 1:r:2]
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
    p, q = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack([p, q], dim=-1).flatten(-2) if case["pairs"] == "near" else torch.cat([p, q], dim=-1)
    return torch.cat([turned, x[..., r:]], dim=-1)


def _plain_heads(st):
    """Normed and rotated queries and keys in 32 bits, [B, N, heads, dim]."""
    case = st["case"]
    at = st["positions"].double()[:, None] + torch.arange(case["tokens"], device="cuda", dtype=torch.float64)
    angle = at[..., None] * st["freqs"]
    return tuple(_rotated(_normed(_heads(st[n], case["dim"]), st[n + "_weight"]), angle, case) for n in "qk")


def _plain_rope(st):
    q, k = (x.flatten(2).to(st["q"].dtype) for x in _plain_heads(st))
    if st["lengths"] is not None:
        valid = (torch.arange(st["case"]["tokens"], device="cuda") < st["lengths"][:, None])[..., None]
        q, k = torch.where(valid, q, 0.0), torch.where(valid, k, 0.0)
    return q, k


def _rows_of(positions, case):
    """[B, held]: the cache's row of each token that a full stream holds, in order."""
    S, W = case["sinks"], case["window"]
    p = positions.long()[:, None]
    return torch.cat([torch.arange(S, device="cuda").expand(len(p), S), S + (p - S + torch.arange(W, device="cuda")) % W], dim=1)


def _plain_read(cache, positions, case):
    """Rows in order, [B, held, kv_heads * dim], keys and values."""
    at, stream = _rows_of(positions, case), torch.arange(case["batch"], device="cuda")[:, None]
    if len(cache) == 2:
        return tuple(c[stream, at] for c in cache)
    # (the heads' rows in the order of tokens: [B, held, heads, dim])
    return tuple((c.transpose(1, 2)[stream, at][..., :case["dim"]].float() * cache[2].transpose(1, 2)[stream, at][..., i, None])
                 .to(DTYPES[case["dtype"]]).flatten(2) for i, c in enumerate(cache[:2]))


def _plain_put(st, k, v):
    """fp32 [B, N, heads, dim] into the cache of 8 bits."""
    case, pos = st["case"], st["positions"].long()
    T, W, S = case["tokens"], case["window"], case["sinks"]
    token = pos[:, None] + torch.arange(T, device="cuda")
    kept = (token < S) | (token >= (pos[:, None] + T - W))
    slot = torch.where(token < S, token, S + (token - S) % W)
    b, t = kept.nonzero(as_tuple=True)
    most = torch.stack([k, v], dim=-1).abs().amax(dim=3)                                  # [B, N, heads, 2]
    st["cache"][2][b, :, slot[b, t]] = (most / 127.0)[b, t]
    k, v = (torch.round(x * 127.0 / most[..., i, None]).to(torch.int8) for i, x in enumerate((k, v)))
    st["cache"][0][b, :, slot[b, t], :case["dim"]] = k[b, t]
    st["cache"][1][b, :, slot[b, t], :case["dim"]] = v[b, t]


def _plain_append(st):
    dim = st["case"]["dim"]
    _plain_put(st, _heads(st["k"], dim), _heads(st["v"], dim))
    return _plain_read(st["cache"], st["after"], st["case"])


def _plain_turn(st):
    q, k = _plain_heads(st)
    _plain_put(st, k, _heads(st["v"], st["case"]["dim"]))
    return q.flatten(2).to(st["q"].dtype), *_plain_read(st["cache"], st["after"], st["case"])


def _plain_attend(st):
    case = st["case"]
    d, G = case["dim"], case["kv_heads"]
    k, v = (c[..., :d].float() * st["cache"][2][..., i, None] for i, c in enumerate(st["cache"][:2]))
    q = _heads(st["q"], d).squeeze(1).unflatten(1, (G, -1))                               # [B, G, r, d]
    seen = torch.arange(k.shape[2], device="cuda") <= st["positions"][:, None]
    s = (q @ k.transpose(-1, -2)) * st["scale"]
    s = torch.where(seen[:, None, None], s, -math.inf)
    p = torch.exp(s - s.amax(dim=-1, keepdim=True))
    out = (p @ v) / p.sum(dim=-1, keepdim=True)
    return out.flatten(1).unsqueeze(1).to(st["q"].dtype)


def run(state):
    st, case = state, state["case"]
    kind = case["kind"]
    if not own:
        if kind == "read":
            return _plain_read(st["cache"], st["positions"], case)
        return {"rope": _plain_rope, "append": _plain_append, "turn": _plain_turn, "attend": _plain_attend}[kind](st)
    from sana_amd import ops
    if kind == "attend":
        return ops.window_attention_q8(st["q"], st["cache"], st["positions"], case["heads"], case["sinks"], scale=st["scale"])
    if kind == "read":
        return ops.window_cache_read(st["cache"], st["positions"], case["sinks"], dim=case["dim"], dtype=DTYPES[case["dtype"]])
    if kind == "rope":
        return ops.qk_norm_rope(st["q"], st["k"], case["heads"], st["q_weight"], st["k_weight"], EPS, st["freqs"],
                                interleaved=case["pairs"] == "near", positions=st["positions"], lengths=st["lengths"])
    if kind == "append":
        ops.window_cache_append_q8_(st["cache"], st["k"], st["v"], st["positions"], case["sinks"])
        return ops.window_cache_read(st["cache"], st["after"], case["sinks"], dim=case["dim"], dtype=st["k"].dtype)
    q, _ = ops.qk_norm_rope_append_q8_(st["q"], st["k"], st["v"], st["cache"], st["positions"], case["heads"], st["q_weight"], st["k_weight"],
                                       EPS, st["freqs"], interleaved=case["pairs"] == "near", sinks=case["sinks"])
    return q, *ops.window_cache_read(st["cache"], st["after"], case["sinks"], dim=case["dim"], dtype=st["k"].dtype)


def exact(case, seed):
    """Stream by stream (attend: head by head too), token by token as complex numbers, in 64 bits."""
    st = prepare(case, seed)
    kind, B, d, G = case["kind"], case["batch"], case["dim"], case["kv_heads"]
    pos = st["positions"].tolist()
    if kind == "attend":
        out = torch.empty(B, 1, case["heads"] * d, dtype=torch.float64, device="cuda")
        for b in range(B):
            held = min(pos[b] + 1, case["sinks"] + case["window"])
            for g in range(G):
                k, v = (st["cache"][i][b, g, :held, :d].double() * st["cache"][2][b, g, :held, i].double()[:, None] for i in (0, 1))
                q = st["q"][b, 0].double().unflatten(0, (G, -1, d))[g]
                out[b, 0].unflatten(0, (G, -1, d))[g] = torch.softmax(q @ k.T * st["scale"], dim=1) @ v
        return out

    def turned(name, b):
        x = st[name][b].double().unflatten(1, (-1, d))
        x = x / (x.square().sum(-1, keepdim=True) / d + EPS).sqrt() * st[name + "_weight"].double()
        r, n = case["rotary"], case["tokens"]
        angle = torch.arange(pos[b], pos[b] + n, device="cuda", dtype=torch.float64)[:, None] * st["freqs"]
        part = x[..., :r].unflatten(-1, (r // 2, 2) if case["pairs"] == "near" else (2, r // 2))
        part = part if case["pairs"] == "near" else part.transpose(-1, -2)
        z = torch.view_as_complex(part.contiguous()) * torch.polar(torch.ones_like(angle), angle)[:, None]
        part = torch.view_as_real(z)
        part = part if case["pairs"] == "near" else part.transpose(-1, -2)
        return torch.cat([part.flatten(-2), x[..., r:]], dim=-1)

    def in_order(b, seen, new):
        """The rows that stream b holds after `seen` tokens, the last of which are `new` [N, heads, d] of keys and of values."""
        S, W, n = case["sinks"], case["window"], 0 if new is None else new[0].shape[0]
        tokens = torch.tensor([*range(S), *range(seen - W, seen)], device="cuda")
        row = torch.where(tokens < S, tokens, S + (tokens - S) % W)
        got = []
        for i in (0, 1):
            if len(st["cache"]) == 2:     # 16 bits: as they are
                got.append(st["cache"][i][b, row].double())
                continue
            x = st["cache"][i][b][:, row, :d].double() * st["cache"][2][b][:, row, i, None].double()     # [heads, held, d]
            x = x.transpose(0, 1)
            late = tokens >= seen - n
            if new is not None and bool(late.any()):
                y = new[i][tokens[late] - (seen - n)]
                most = y.abs().amax(-1, keepdim=True)
                x[late] = torch.round(127 * y / most) * (most / 127)
            got.append(x.flatten(1))
        return got

    if kind == "rope":
        outs = []
        for name in "qk":
            rows = [turned(name, b).flatten(1) for b in range(B)]
            for b in range(B):
                if st["lengths"] is not None:
                    rows[b][int(st["lengths"][b]):] = 0
            outs.append(torch.stack(rows))
        return tuple(outs)
    n = case.get("tokens", 0) if kind != "read" else 0
    held = []
    for b in range(B):
        new = None
        if kind != "read":
            new = (turned("k", b) if kind == "turn" else st["k"][b].double().unflatten(1, (G, d)), st["v"][b].double().unflatten(1, (G, d)))
        held.append(in_order(b, pos[b] + n, new))
    k, v = (torch.stack([x[i] for x in held]) for i in (0, 1))
    return (torch.stack([turned("q", b).flatten(1) for b in range(B)]), k, v) if kind == "turn" else (k, v)


def _kept(case):
    """Tokens of the call that stay in the cache, all streams."""
    return sum(sum(1 for t in range(p, p + case["tokens"]) if t < case["sinks"] or t >= p + case["tokens"] - case["window"])
               for p in _positions(case))


def work(case):
    B, G, d, kind = case["batch"], case["kv_heads"], case["dim"], case["kind"]
    H = case.get("heads", 0)
    if kind == "rope":
        values = sum(_lengths(case)) * (H + G) * d
        return {"bytes": 2 * 2 * values, "flops": 10 * values}
    held = case["sinks"] + case["window"]
    row = 2 * G * (d + 4)      # a token's key and value in 8 bits with their scales
    if kind == "attend":
        seen = sum(min(p + 1, held) for p in _positions(case))
        return {"bytes": row * seen + 2 * 2 * B * H * d, "flops": 4 * d * H * seen}
    in_order = 2 * 2 * B * held * G * d
    if kind == "read":
        return {"bytes": (in_order if case["bits"] == 16 else row * B * held) + in_order, "flops": 0 if case["bits"] == 16 else 2 * B * held * G * d}
    kept = _kept(case)         # their rows in, their codes out, the codes of the others in, all rows in order out
    bytes_ = 2 * 2 * kept * G * d + row * kept + row * (B * held - kept) + in_order
    flops = 2 * 3 * kept * G * d + 2 * B * held * G * d
    if kind == "turn":
        bytes_ += 2 * 2 * B * case["tokens"] * H * d
        flops += 10 * (B * case["tokens"] * H + kept * G) * d
    return {"bytes": bytes_, "flops": flops}
