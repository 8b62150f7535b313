"""Causal token mixing whose memory does not grow with the stream, as cases that can be timed and compared.

A case is a dict of plain values.  ``listed()`` names the ones that are always looked at, ``draw(rng)`` makes more of the
same ranges, ``prepare`` builds what a program holds before the call, ``run`` makes one pass (the framework's kernels where
``own`` is true, elementary torch operations in 32 bits where it is not), ``exact`` is the same in 64 bits from the
definition, and ``work`` says what the pass cannot do without.

Four kinds of work, on the token-major rows that a fused projection leaves (q, k and v are views of one tensor):

* ``decay``   linear attention with a decay for each head.  State S [d of v][d of k] per head,
              S_t = exp(g_h) S_{t-1} + v_t k_t^T,   o_t = scale * S_t q_t;
              a prompt of many tokens, or one token of each stream; from an empty state or one that is carried,
* ``window``  softmax attention in which a query sees the last ``window`` keys up to its own and the first ``sinks`` keys;
              the queries are the last tokens of the keys,
* ``append``  the keys and values of new tokens go into a cache that holds the sinks and, as a ring, the last ``window`` others,
* ``step``    one new token of each stream: into the cache, and its attention over what the cache then holds.

Widths are those of the image and video models here (1152 and 2240 channels, heads of 32, 72 and 112) and generic ones (heads of 64, 96
and 128); 1560 tokens are a latent frame of 480p, 4680 the three frames of a streamed chunk.
"""
import math

import torch

own = False
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
BLOCK = 256      # tokens that the plain decay form takes at a time
QUERIES = 1024   # queries that the plain window form takes at a time


def _decay(name, batch, tokens, heads, dim, *, dtype="bf16", carried=False, ragged=False):
    return {"name": name, "kind": "decay", "batch": batch, "tokens": tokens, "heads": heads, "dim": dim, "dtype": dtype,
            "carried": carried, "ragged": ragged}


def _window(name, batch, tokens, heads, kv_heads, dim, window, sinks, *, past=0, dtype="bf16", ragged=False):
    return {"name": name, "kind": "window", "batch": batch, "tokens": tokens, "past": past, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "window": window, "sinks": sinks, "dtype": dtype, "ragged": ragged}


def _cached(name, kind, batch, tokens, heads, kv_heads, dim, window, sinks, *, dtype="bf16"):
    return {"name": name, "kind": kind, "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "window": window, "sinks": sinks, "dtype": dtype}


def listed():
    return [
        # one stream, one token, at the width of the large image model: nothing but latency
        _decay("decay_token_b1", 1, 1, 20, 112, carried=True),
        # a full serving batch, a token of each stream: the states are read and written once
        _decay("decay_token_b128", 128, 1, 35, 64, carried=True),
        # a short prompt in half precision: a few chunks
        _decay("decay_prompt_300_fp16", 1, 300, 70, 32, dtype="fp16"),
        # the next three frames of two streams of unlike length
        _decay("decay_chunk_b2", 2, 4680, 20, 112, carried=True, ragged=True),
        # the whole of a 480p clip of 21 latent frames in one go: long, and few heads
        _decay("decay_clip_21f", 1, 32760, 20, 112),
        # a short prompt over a window that it does not fill
        _window("window_prompt_200", 1, 200, 16, 16, 72, 256, 4),
        # three streamed frames behind six of the past and the first frame, which stays; shared key heads, half precision
        _window("window_chunk_gqa_fp16", 2, 4680, 20, 5, 112, 9360, 1560, past=10920, dtype="fp16"),
        # the tokens of one large image in scan order
        _window("window_16384", 1, 16384, 20, 20, 112, 4096, 64),
        # a streamed chunk goes into the caches of two streams
        _cached("append_chunk_b2", "append", 2, 4680, 20, 20, 112, 9360, 1560),
        # the last tokens of a batch of long prompts go into short caches
        _cached("append_prompts_b16", "append", 16, 4096, 16, 4, 128, 2048, 4),
        # one stream, one token over a short window
        _cached("step_b1", "step", 1, 1, 16, 16, 72, 1024, 4),
        # a full serving batch over long windows with shared key heads
        _cached("step_gqa_b64", "step", 64, 1, 32, 8, 128, 8192, 4),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["decay", "token", "window", "append", "step"])
    dtype = rng.choice(["bf16", "fp16"])
    heads, dim = rng.choice([(36, 32), (70, 32), (35, 64), (16, 72), (12, 96), (20, 112), (16, 128)])
    if kind == "token":
        return {"kind": "decay", "batch": _log_int(rng, 1, 192), "tokens": 1, "heads": heads, "dim": dim, "dtype": dtype,
                "carried": True, "ragged": False}
    if kind == "decay":
        tokens = _log_int(rng, 2, 24000)
        return {"kind": "decay", "batch": rng.randint(1, max(1, min(16, 32000 // tokens))), "tokens": tokens, "heads": heads,
                "dim": dim, "dtype": dtype, "carried": rng.random() < 0.5, "ragged": rng.random() < 0.5}
    kv_heads = heads // rng.choice([g for g in (1, 2, 4, 5, 7, 8) if heads % g == 0])
    window, sinks = _log_int(rng, 16, 6000), rng.choice([0, 1, 4, 64, 390])
    common = {"heads": heads, "kv_heads": kv_heads, "dim": dim, "window": window, "sinks": sinks, "dtype": dtype}
    if kind == "window":
        tokens = _log_int(rng, 2, 8000)
        return {"kind": kind, "batch": rng.randint(1, max(1, min(4, 8000 // tokens))), "tokens": tokens,
                "past": rng.choice([0, 0, sinks + window, rng.randint(1, 5000)]), "ragged": rng.random() < 0.4, **common}
    tokens = 1 if kind == "step" else _log_int(rng, 1, 6000)
    return {"kind": kind, "batch": _log_int(rng, 1, 48), "tokens": tokens, **common}


def _spread(count, lo, hi):
    """`count` whole numbers from lo to hi, evenly spread, hi among them."""
    return [hi - (hi - lo) * i // max(1, count - 1) for i in range(count)]


def _lengths(case):
    n = case["tokens"]
    return _spread(case["batch"], n // 2, n) if case.get("ragged") else [n] * case["batch"]


def _positions(case):
    """Tokens that each stream has seen before: from a part of what its cache holds to three times that."""
    full = case["sinks"] + case["window"]
    return _spread(case["batch"], full // 2, 3 * full) if case["batch"] > 1 else [2 * full + 7]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt, B, T, H, d = DTYPES[case["dtype"]], case["batch"], case["tokens"], case["heads"], case["dim"]
    order = torch.randperm(B, generator=gen, device="cuda").cpu()

    def rows(values):
        return torch.tensor(values)[order].to(device="cuda", dtype=torch.int32)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dt)

    st = {"case": case, "scale": d ** -0.5}
    if case["kind"] == "decay":
        qkv = normal(B, T, 3 * H * d)
        st["q"], st["k"], st["v"] = qkv.split(H * d, dim=2)
        # half-lives from some five tokens to some three thousand
        st["log_decay"] = torch.log1p(-torch.exp2(-torch.linspace(3.0, 12.0, H, device="cuda")))
        st["state"] = torch.randn((B, H, d, d), generator=gen, device="cuda") if case["carried"] else None
        st["lengths"] = rows(_lengths(case)) if case["ragged"] else None
        st["state_out"] = torch.empty(B, H, d, d, device="cuda") if case["carried"] else None   # the program's second buffer
        return st
    G = case["kv_heads"]
    if case["kind"] == "window":
        qkv = normal(B, case["past"] + T, (H + 2 * G) * d)
        q, st["k"], st["v"] = qkv.split([H * d, G * d, G * d], dim=2)
        st["q"] = q[:, case["past"]:]
        st["lengths"] = rows(_lengths(case)) if case["ragged"] else None
        return st
    qkv = normal(B, T, (H + 2 * G) * d)
    st["q"], st["k"], st["v"] = qkv.split([H * d, G * d, G * d], dim=2)
    held = case["sinks"] + case["window"]
    st["cache_k"], st["cache_v"] = normal(B, held, G * d), normal(B, held, G * d)
    st["positions"] = rows(_positions(case))
    return st


def _heads(t, heads):
    """[B, N, heads * d] -> fp32 [B, heads, N, d]"""
    return t.unflatten(2, (heads, -1)).transpose(1, 2).float()


def _rows_of(t, dtype):
    """[B, heads, N, d] -> [B, N, heads * d]"""
    return t.transpose(1, 2).flatten(2).to(dtype)


def _valid(st, tokens):
    """[B, tokens]: the tokens that a stream has, or None where it has all."""
    return None if st["lengths"] is None else torch.arange(tokens, device="cuda") < st["lengths"][:, None]


def _plain_decay(st):
    case, g = st["case"], st["log_decay"].double()
    B, T, H, d = case["batch"], case["tokens"], case["heads"], case["dim"]
    q, k, v = (_heads(st[n], H) for n in "qkv")
    valid = _valid(st, T)
    if valid is not None:
        k, v = k * valid[:, None, :, None], v * valid[:, None, :, None]
    # blocks of tokens: within a block by its scores, across blocks by the states in front of them
    C = min(BLOCK, T)
    nb = -(-T // C)
    pad = nb * C - T
    qb, kb, vb = (torch.nn.functional.pad(t, (0, 0, 0, pad)).unflatten(2, (nb, C)) for t in (q, k, v))
    at = torch.arange(C, device="cuda", dtype=torch.float64)
    apart = at[:, None] - at[None, :]
    D = torch.where(apart >= 0, torch.exp(apart.clamp(min=0) * g[:, None, None]), 0.0).float()            # [H, C, C]
    to_end = torch.exp((C - 1 - at) * g[:, None]).float()                                                # [H, C]
    within = ((qb @ kb.transpose(-1, -2)) * D[:, None]) @ vb
    ends = (vb * to_end[:, None, :, None]).transpose(-1, -2) @ kb                                         # [B, H, nb, dv, dk]
    block = torch.arange(nb, device="cuda", dtype=torch.float64)
    gap = block[:, None] - 1 - block[None, :]
    carry = torch.where(gap >= 0, torch.exp(gap.clamp(min=0) * C * g[:, None, None]), 0.0).float()         # [H, nb, nb]
    before = (carry @ ends.flatten(3)).unflatten(3, (d, d))
    if st["state"] is not None:
        before = before + torch.exp(block * C * g[:, None]).float()[:, :, None, None] * st["state"][:, :, None]
    from_start = torch.exp((at + 1) * g[:, None]).float()
    across = (qb @ before.transpose(-1, -2)) * from_start[:, None, :, None]
    out = ((within + across) * st["scale"]).flatten(2, 3)[:, :, :T]
    if valid is not None:
        out = torch.where(valid[:, None, :, None], out, 0.0)
    count = st["lengths"].double() if valid is not None else torch.full((B,), float(T), device="cuda", dtype=torch.float64)
    age = (count[:, None] - 1 - torch.arange(T, device="cuda")).clamp(min=0)                              # [B, T]
    w = torch.exp(age[:, None] * g[:, None]).float()                                                      # [B, H, T]
    state = (v * w[..., None]).transpose(-1, -2) @ k
    if st["state"] is not None:
        state = state + torch.exp(count[:, None] * g).float()[..., None, None] * st["state"]
    return _rows_of(out, st["q"].dtype), state


def _plain_window(st):
    case = st["case"]
    B, T, H, G, W, S = (case[n] for n in ("batch", "tokens", "heads", "kv_heads", "window", "sinks"))
    past, r = case["past"], case["heads"] // case["kv_heads"]
    q, k, v = _heads(st["q"], H), _heads(st["k"], G), _heads(st["v"], G)
    Q = min(QUERIES, T)
    nb = -(-T // Q)
    q = torch.nn.functional.pad(q, (0, 0, 0, nb * Q - T)).unflatten(2, (nb, Q)).unflatten(1, (G, r))       # [B, G, r, nb, Q, d]
    # a block of queries against the sinks and the band of keys that any of them can see
    first = past + torch.arange(nb, device="cuda") * Q
    band = first[:, None] - (W - 1) + torch.arange(W - 1 + Q, device="cuda")                              # [nb, W - 1 + Q]
    sink = torch.arange(S, device="cuda").expand(nb, S)
    key = torch.cat([sink, band], dim=1)
    query = first[:, None] + torch.arange(Q, device="cuda")
    apart = query[:, :, None] - key[:, None, :]
    seen = (apart >= 0) & (key[:, None, :] >= 0)
    in_band = torch.arange(key.shape[1], device="cuda") >= S
    # in the band what the window holds and is no sink; among the sinks all up to the query
    seen &= torch.where(in_band, (apart < W) & (key[:, None, :] >= S), True)
    at = key.clamp(0, past + T - 1)
    kb, vb = (t[:, :, at][:, :, None] for t in (k, v))                                                    # [B, G, 1, nb, keys, d]
    scores = (q @ kb.transpose(-1, -2)) * st["scale"]
    scores = torch.where(seen, scores, -math.inf)
    p = torch.exp(scores - scores.amax(dim=-1, keepdim=True))
    out = (p @ vb) / p.sum(dim=-1, keepdim=True)
    out = out.flatten(3, 4).flatten(1, 2)[:, :, :T]
    valid = _valid(st, T)
    if valid is not None:
        out = torch.where(valid[:, None, :, None], out, 0.0)
    return _rows_of(out, st["q"].dtype)


def _plain_append(st):
    case, pos = st["case"], st["positions"].long()
    T, W, S = case["tokens"], case["window"], case["sinks"]
    token = pos[:, None] + torch.arange(T, device="cuda")
    kept = (token < S) | (token >= (pos[:, None] + T - W))
    slot = torch.where(token < S, token, S + (token - S) % W)
    b, t = kept.nonzero(as_tuple=True)
    st["cache_k"][b, slot[b, t]] = st["k"][b, t]
    st["cache_v"][b, slot[b, t]] = st["v"][b, t]
    return st["cache_k"], st["cache_v"]


def _plain_step(st):
    case, pos = st["case"], st["positions"].long()
    B, H, G, W, S = (case[n] for n in ("batch", "heads", "kv_heads", "window", "sinks"))
    slot = torch.where(pos < S, pos, S + (pos - S) % W)
    stream = torch.arange(B, device="cuda")
    st["cache_k"][stream, slot] = st["k"][:, 0]
    st["cache_v"][stream, slot] = st["v"][:, 0]
    q = _heads(st["q"], H).unflatten(1, (G, H // G)).squeeze(3)                                            # [B, G, r, d]
    k, v = _heads(st["cache_k"], G), _heads(st["cache_v"], G)
    seen = torch.arange(S + W, device="cuda") <= pos[:, None]
    scores = (q @ k.transpose(-1, -2)) * st["scale"]
    scores = torch.where(seen[:, None, None], scores, -math.inf)
    p = torch.exp(scores - scores.amax(dim=-1, keepdim=True))
    out = (p @ v) / p.sum(dim=-1, keepdim=True)
    return out.flatten(1).unsqueeze(1).to(st["q"].dtype), st["cache_k"], st["cache_v"]


def run(state):
    st, case = state, state["case"]
    if not own:
        return {"decay": _plain_decay, "window": _plain_window, "append": _plain_append, "step": _plain_step}[case["kind"]](st)
    from sana_amd import ops
    if case["kind"] == "decay":
        return ops.decay_linear_attention(st["q"], st["k"], st["v"], st["log_decay"], scale=st["scale"], state=st["state"],
                                          lengths=st["lengths"], state_out=st["state_out"])
    if case["kind"] == "window":
        return ops.window_attention(st["q"], st["k"], st["v"], case["heads"], case["window"], case["sinks"], scale=st["scale"],
                                    lengths=st["lengths"])
    if case["kind"] == "append":
        ops.window_cache_append_(st["cache_k"], st["cache_v"], st["k"], st["v"], st["positions"], case["sinks"])
        return st["cache_k"], st["cache_v"]
    out = ops.window_attention_step_(st["q"], st["k"], st["v"], st["cache_k"], st["cache_v"], st["positions"], case["heads"],
                                     case["sinks"], scale=st["scale"])
    return out, st["cache_k"], st["cache_v"]


def exact(case, seed):
    """Head by head, every query against every key, in 64 bits."""
    st = prepare(case, seed)
    if case["kind"] == "append":
        return None
    B, T, H, d = case["batch"], case["tokens"], case["heads"], case["dim"]
    G, scale = case.get("kv_heads", H), st["scale"]
    out = torch.zeros(B, T, H * d, dtype=torch.float64, device="cuda")
    head = lambda name, b, h: st[name][b, :, h * d:(h + 1) * d].double()  # noqa: E731
    if case["kind"] == "decay":
        final = torch.empty(B, H, d, d, dtype=torch.float64, device="cuda")
        for b in range(B):
            n = T if st["lengths"] is None else int(st["lengths"][b])
            i = torch.arange(n, device="cuda", dtype=torch.float64)
            for h in range(H):
                rate = float(st["log_decay"][h].double())
                q, k, v = (head(name, b, h)[:n] for name in "qkv")
                weight = (i[:, None] - i[None, :]).mul_(rate).exp_().tril_()
                o = weight.mul_(q @ k.T) @ v
                del weight
                s = v.T @ (k * torch.exp(rate * (n - 1 - i))[:, None])
                if st["state"] is not None:
                    s0 = st["state"][b, h].double()
                    o += torch.exp(rate * (i + 1))[:, None] * (q @ s0.T)
                    s += math.exp(rate * n) * s0
                out[b, :n, h * d:(h + 1) * d] = scale * o
                final[b, h] = s
        return out, final
    if case["kind"] == "window":
        keys = case["past"] + T
        i = torch.arange(case["past"], keys, device="cuda")[:, None]
        j = torch.arange(keys, device="cuda")[None, :]
        hidden = (j > i) | ((i - j >= case["window"]) & (j >= case["sinks"]))
        for b in range(B):
            n = T if st["lengths"] is None else int(st["lengths"][b])
            for h in range(H):
                s = head("q", b, h) @ head("k", b, h * G // H).T * scale
                p = s.masked_fill_(hidden, -math.inf).softmax(dim=1)
                out[b, :n, h * d:(h + 1) * d] = (p @ head("v", b, h * G // H))[:n]
        return out
    # the step: the cache as the tokens that it holds, oldest first
    window, sinks = case["window"], case["sinks"]
    for b in range(B):
        p = int(st["positions"][b])
        held = list(range(min(p + 1, sinks))) + list(range(max(sinks, p + 1 - window), p + 1))
        at = torch.tensor([t if t < sinks else sinks + (t - sinks) % window for t in held], device="cuda")
        for g in range(G):
            k, v = st["cache_k"][b, :, g * d:(g + 1) * d].double()[at], st["cache_v"][b, :, g * d:(g + 1) * d].double()[at]
            k[-1], v[-1] = head("k", b, g)[0], head("v", b, g)[0]
            for h in range(g * H // G, (g + 1) * H // G):
                out[b, 0, h * d:(h + 1) * d] = torch.softmax(k @ head("q", b, h)[0] * scale, dim=0) @ v
    return out, None, None


def _pairs(case, lengths):
    """Query-key pairs that are looked at, all streams, one head."""
    past, W, S = case["past"], case["window"], case["sinks"]
    return sum(min(W, p + 1) + max(0, min(S, p + 1 - W)) for n in lengths for p in range(past, past + n))


def work(case):
    B, T, H, d = case["batch"], case["tokens"], case["heads"], case["dim"]
    G = case.get("kv_heads", H)
    if case["kind"] == "decay":
        tokens = sum(_lengths(case))
        states = (2 if case["carried"] else 1) * B * H * d * d * 4
        return {"bytes": 4 * 2 * tokens * H * d + states, "flops": 4 * tokens * H * d * d}
    if case["kind"] == "window":
        lengths = _lengths(case)
        keys = sum(min(case["past"], case["sinks"] + case["window"] - 1) + n for n in lengths)
        return {"bytes": 2 * (2 * sum(lengths) * H * d + 2 * keys * G * d), "flops": 4 * d * H * _pairs(case, lengths)}
    if case["kind"] == "append":
        kept = sum(sum(1 for t in range(p, p + T) if t < case["sinks"] or t >= p + T - case["window"]) for p in _positions(case))
        return {"bytes": 2 * 2 * 2 * kept * G * d, "flops": 0}
    held = sum(min(p + 1, case["sinks"] + case["window"]) for p in _positions(case))
    return {"bytes": 2 * (2 * held * G * d + 2 * B * H * d + 2 * B * G * d), "flops": 4 * d * H * held}
