"""Operators around the decoder - rotary positions, a key / value cache held in 4 bits, scores of given tokens - as cases
that can be timed, each with a plain form in elementary torch operations.

Sizes are those of the two architectures that the tests and bench.py run (20 query / 5 key heads of 128 and a vocabulary of
128256; 64 / 8 heads), context lengths from one token to 131072, and generic ones around them.

Kinds of case:
  rotate    queries and keys of a step or a prompt turned by their positions; "grad": with the gradient
  append    new tokens rotated and written into a 4-bit cache; what is written is read back as the values it stands for
  attend    attention of new tokens over a 4-bit cache that holds them already
  logprobs  log probabilities of given tokens, entropy and the most probable alternatives; "grad": with the gradient
"""
import math

import torch

DEV = "cuda"
VOCAB = 128256
GROUP = 32                     # values that share a scale in the 4-bit cache
own = False                    # True: the framework's operators, False: the plain forms


def listed():
    return [
        # one token for each of eight sequences: latency
        dict(name="rotate_step", kind="rotate", batch=8, tokens=1, heads=20, kv_heads=5, dim=128, rotary=128, half=False,
             scaling="none", max_len=2048, dtype="bfloat16", grad=False),
        # prompts of the wide model, half layout, at positions that a scaled table reaches
        dict(name="rotate_prompt", kind="rotate", batch=2, tokens=2048, heads=64, kv_heads=8, dim=128, rotary=128, half=True,
             scaling="yarn", max_len=131072, dtype="bfloat16", grad=False),
        # a training batch of odd length: part of the head rotated, fp32, forward and backward
        dict(name="rotate_grad", kind="rotate", batch=4, tokens=1023, heads=20, kv_heads=5, dim=128, rotary=64, half=True,
             scaling="linear", max_len=4096, dtype="float32", grad=True),
        # one new token for each of eight sequences of different length
        dict(name="append_step", kind="append", batch=8, tokens=1, heads=20, kv_heads=5, dim=128, max_len=2048, padded=False),
        # three prompts padded to the longest
        dict(name="append_prompt", kind="append", batch=3, tokens=1226, heads=20, kv_heads=5, dim=128, max_len=2048, padded=True),
        # interactive decoding, one sequence
        dict(name="attend_step", kind="attend", batch=1, tokens=1, heads=20, kv_heads=5, dim=128, past=600, max_len=2048, window=0),
        # batched decoding with the wide model's heads, sequences of up to 8000 tokens
        dict(name="attend_batch", kind="attend", batch=32, tokens=1, heads=64, kv_heads=8, dim=128, past=8000, max_len=8192, window=0),
        # one sequence over a very long document
        dict(name="attend_long", kind="attend", batch=1, tokens=1, heads=20, kv_heads=5, dim=128, past=131000, max_len=131072, window=0),
        # the second chunk of a long prompt
        dict(name="attend_chunk", kind="attend", batch=1, tokens=2048, heads=20, kv_heads=5, dim=128, past=2048, max_len=4096, window=0),
        # scores beside three generated tokens
        dict(name="logprobs_step", kind="logprobs", rows=3, vocab=VOCAB, top=5, dtype="float32", grad=False),
        # scoring two texts of 613 tokens
        dict(name="logprobs_prompt", kind="logprobs", rows=1226, vocab=VOCAB, top=20, dtype="bfloat16", grad=False),
        # policy gradient with an entropy term
        dict(name="logprobs_grad", kind="logprobs", rows=512, vocab=VOCAB, top=0, dtype="float32", grad=True),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["rotate", "append", "attend", "attend", "attend", "logprobs", "logprobs"])
    kv_heads = rng.choice([1, 2, 5, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 8])
    dim = rng.choice([64, 128, 128])
    if kind == "rotate":
        batch = rng.randint(1, 8)
        tokens = _log(rng, 1, 4096 // batch)
        return dict(kind=kind, batch=batch, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, rotary=rng.choice([dim, dim // 2, 40]),
                    half=rng.random() < 0.5, scaling=rng.choice(["none", "linear", "ntk", "yarn", "wavelength"]),
                    max_len=_log(rng, max(64, tokens), 131072), dtype=rng.choice(["bfloat16", "float16", "float32"]), grad=rng.random() < 0.4)
    if kind == "append":
        batch = rng.randint(1, 16)
        tokens = _log(rng, 1, 4096 // batch)
        return dict(kind=kind, batch=batch, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, max_len=tokens + _log(rng, 1, 2048),
                    padded=rng.random() < 0.5)
    if kind == "attend":
        tokens = 1 if rng.random() < 0.6 else _log(rng, 2, 800)
        past = _log(rng, 1, min(4000, 120000000 // (tokens * heads) - tokens) if tokens > 1 else 60000)
        batch = min(rng.randint(1, 48), max(1, (12000000 if tokens == 1 else 120000000 // tokens) // ((past + tokens) * heads)))
        return dict(kind=kind, batch=batch, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, past=past, max_len=past + tokens + rng.randint(0, 500),
                    window=0 if rng.random() < 0.7 else _log(rng, 16, 2000))
    grad = rng.random() < 0.4
    vocab = _log(rng, 300, 200000)
    return dict(kind=kind, rows=_log(rng, 1, max(1, (60000000 if grad else 120000000) // vocab)), vocab=vocab,
                top=0 if grad else rng.choice([0, 1, 5, 20, 32]), dtype=rng.choice(["float32", "bfloat16", "float16"]), grad=grad)


# ---------------------------------------------------------------------------------------------- the pieces of the plain forms

SCALING = {"none": None, "linear": dict(type="linear", factor=4.0), "ntk": dict(type="ntk", factor=4.0),
           "yarn": dict(type="yarn", factor=16.0, original_len=8192, beta_fast=32.0, beta_slow=1.0),
           "wavelength": dict(type="wavelength", factor=8.0, original_len=8192, low=1.0, high=4.0)}
THETA = 500000.0


def angles(rotary, scaling):
    """Angle per position of every pair, in 64 bits, and the factor of cosines and sines."""
    pair = torch.arange(0, rotary, 2, dtype=torch.float64, device=DEV)
    inv = THETA ** (-pair / rotary)
    if scaling == "none":
        return inv, 1.0
    s = SCALING[scaling]
    if scaling == "linear":
        return inv / s["factor"], 1.0
    if scaling == "ntk":
        return (THETA * s["factor"] ** (rotary / (rotary - 2))) ** (-pair / rotary), 1.0
    if scaling == "yarn":
        def at(turns):         # index of the pair that turns so often over the original length
            return rotary * math.log(s["original_len"] / (turns * 2 * math.pi)) / (2 * math.log(THETA))
        lo, hi = max(math.floor(at(s["beta_fast"])), 0), min(math.ceil(at(s["beta_slow"])), rotary - 1)
        slow = ((pair / 2 - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return inv * (1 - slow) + inv / s["factor"] * slow, 0.1 * math.log(s["factor"]) + 1
    turns = s["original_len"] * inv / (2 * math.pi)
    keep = ((turns - s["low"]) / (s["high"] - s["low"])).clamp(0, 1)
    return inv * keep + inv / s["factor"] * (1 - keep), 1.0


def tables(max_len, rotary, scaling):
    inv, factor = angles(rotary, scaling)
    a = torch.arange(max_len, dtype=torch.float64, device=DEV)[:, None] * inv
    return (a.cos() * factor).float(), (a.sin() * factor).float()


def turn(x, cos, sin, half, back=False):
    """x [B, T, H, D] turned by cos, sin [B, T, rotary / 2]; 32 bits, rounded once."""
    n = cos.shape[-1]
    c, s = cos[:, :, None], -sin[:, :, None] if back else sin[:, :, None]
    f = x[..., : 2 * n].float()
    a, b = (f[..., :n], f[..., n:]) if half else (f[..., 0::2], f[..., 1::2])
    p, q = a * c - b * s, a * s + b * c
    y = torch.cat([p, q], -1) if half else torch.stack([p, q], -1).flatten(-2)
    return torch.cat([y.to(x.dtype), x[..., 2 * n:]], -1)


def quantise(x):
    """codes 0 .. 15 and fp16 scales of [..., D]: the scale takes a group's value of largest magnitude to code 0."""
    g = x.float().unflatten(-1, (-1, GROUP))
    hi, lo = g.amax(-1), g.amin(-1)
    scale = (torch.where(hi >= -lo, hi, lo) / -8).to(torch.float16)
    s = scale.float()[..., None]
    code = torch.where(s == 0, torch.full_like(g, 8.0), (g / s).round() + 8).clamp(0, 15)
    return code.flatten(-2).to(torch.uint8), scale


def pack(code, unit):
    """Two codes a byte; the groups' units of `unit` bytes in turn, as a row of the cache holds them."""
    b = code[..., 0::2] | code[..., 1::2] << 4
    return b.unflatten(-1, (code.shape[-1] // GROUP, 16 // unit, unit)).transpose(-3, -2).flatten(-3).contiguous()


def unpack(b, unit):
    b = b.unflatten(-1, (16 // unit, b.shape[-1] // 16, unit)).transpose(-3, -2).flatten(-3)
    return torch.stack([b & 15, b >> 4], -1).flatten(-2)


K_UNIT, V_UNIT = 4, 2


def values(code, scale):
    return ((code.float() - 8).unflatten(-1, (-1, GROUP)) * scale.float()[..., None]).flatten(-2)


def new_cache(batch, kv_heads, max_len, dim):
    """Codes and scales of keys, then of values; room for whole tiles of 64 tokens."""
    return [torch.zeros((batch, kv_heads, (max_len + 63) // 64 * 64, n), dtype=t, device=DEV)
            for n, t in ((dim // 2, torch.uint8), (dim // GROUP, torch.float16)) * 2]


# ---------------------------------------------------------------------------------------------- cases

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def prepare(case, seed):
    g = _gen(seed)
    kind = case["kind"]

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEV)

    if kind == "logprobs":
        # logits of a language model: a broad bulk and a few tokens that stand out; a twentieth of the vocabulary is banned
        x = 2.5 * normal(case["rows"], case["vocab"])
        x += 6 * (torch.rand(x.shape, generator=g, device=DEV) < 2e-4)
        banned = torch.rand(case["vocab"], generator=g, device=DEV) < 0.05
        targets = torch.randint(0, case["vocab"], (case["rows"],), generator=g, device=DEV)
        banned[targets] = False
        if not case["grad"]:
            x.masked_fill_(banned, -math.inf)
        st = dict(case=case, logits=x.to(getattr(torch, case["dtype"])), targets=targets)
        if case["grad"]:
            st["grad_logprob"], st["grad_entropy"] = normal(case["rows"]), 0.1 * normal(case["rows"])
            if own:
                st["logits"].requires_grad_()
        return st

    B, T, H, K, D = (case[n] for n in ("batch", "tokens", "heads", "kv_heads", "dim"))
    if kind == "rotate":
        st = dict(case=case)
        qkv = normal(B, T, H + 2 * K, D).to(getattr(torch, case["dtype"]))       # the projections of one linear: views into it
        first = torch.randint(0, case["max_len"] - T + 1, (B, 1), generator=g, device=DEV)
        st["positions"] = first + torch.arange(T, device=DEV)
        st["q"], st["k"] = qkv[:, :, :H], qkv[:, :, H: H + K]
        if case["grad"]:
            st["gq"], st["gk"] = normal(B, T, H, D).to(qkv.dtype), normal(B, T, K, D).to(qkv.dtype)
            if own:
                st["q"], st["k"] = st["q"].detach().requires_grad_(), st["k"].detach().requires_grad_()
        if own:
            from ternainfer_b200.rotary import rotary_table
            st["table"] = rotary_table(D, case["max_len"], THETA, rotary_dim=case["rotary"], layout="half" if case["half"] else "interleaved",
                                       scaling=SCALING[case["scaling"]], device=DEV)
        else:
            st["cos"], st["sin"] = tables(case["max_len"], case["rotary"], case["scaling"])
        return st

    if kind == "append":
        cache = new_cache(B, K, case["max_len"], D)
        qkv = normal(B, T, H + 2 * K, D).to(torch.bfloat16)
        st = dict(case=case, cache=cache, q=qkv[:, :, :H], k=qkv[:, :, H: H + K], v=qkv[:, :, H + K:],
                  start=torch.randint(0, case["max_len"] - T + 1, (B,), generator=g, device=DEV),
                  counts=torch.randint(max(1, T // 2), T + 1, (B,), generator=g, device=DEV) if case["padded"] else None)
        if own:
            from ternainfer_b200.kv4 import KV4Cache
            from ternainfer_b200.rotary import rotary_table
            st["cache"], st["table"] = KV4Cache(*cache), rotary_table(D, case["max_len"], THETA, device=DEV)
        else:
            st["cos"], st["sin"] = tables(case["max_len"], D, "none")
        return st

    # attend: keys with a few strong channels, as rotated keys have them; sequences of between half of `past` and all of it
    start = torch.randint((case["past"] + 1) // 2, case["past"] + 1, (B,), generator=g, device=DEV)
    if B == 1:
        start.fill_(case["past"])
    strong = 1 + 2 * (torch.rand((K, 1, D), generator=g, device=DEV) < 0.05)
    cache = new_cache(B, K, case["max_len"], D)
    for b in range(B):
        for unit, at, scale in ((K_UNIT, 0, strong), (V_UNIT, 2, 1.0)):
            code, s = quantise((normal(K, cache[at].shape[2], D) * scale).to(torch.bfloat16))
            cache[at][b], cache[at + 1][b] = pack(code, unit), s
    q = (1.5 * normal(B, T, H, D)).to(torch.bfloat16)
    if own:
        from ternainfer_b200.kv4 import KV4Cache
        cache = KV4Cache(*cache)
    return dict(case=case, cache=cache, q=q, start=start)


def run(state):
    case = state["case"]
    return globals()[("own_" if own else "plain_") + case["kind"]](state, case)


def plain_rotate(st, case):
    c, s = st["cos"][st["positions"]], st["sin"][st["positions"]]
    out = [turn(st["q"], c, s, case["half"]), turn(st["k"], c, s, case["half"])]
    return out + [turn(st["gq"], c, s, case["half"], back=True), turn(st["gk"], c, s, case["half"], back=True)] if case["grad"] else out


def own_rotate(st, case):
    from ternainfer_b200.rotary import rotate
    q, k = rotate(st["q"], st["k"], st["table"], st["positions"])
    if case["grad"]:
        gq, gk = torch.autograd.grad((q, k), (st["q"], st["k"]), (st["gq"], st["gk"]))
        return [q, k, gq, gk]
    return [q, k]


def plain_append(st, case):
    B, T = case["batch"], case["tokens"]
    at = st["start"][:, None] + torch.arange(T, device=DEV)
    new = torch.ones((B, T), dtype=torch.bool, device=DEV) if st["counts"] is None else torch.arange(T, device=DEV) < st["counts"][:, None]
    c, s = st["cos"][at], st["sin"][at]
    q, k = turn(st["q"], c, s, False), turn(st["k"], c, s, False)
    b = torch.arange(B, device=DEV)[:, None].expand(B, T)
    for x, unit, i in ((k, K_UNIT, 0), (st["v"], V_UNIT, 2)):
        code, scale = quantise(x)
        for to, row in ((st["cache"][i], pack(code, unit)), (st["cache"][i + 1], scale)):
            to[b, :, at] = torch.where(new[..., None, None], row, to[b, :, at])
    # what the cache stands for in the rows of these tokens; zeros in the rows behind a sequence's last token
    back = [values(unpack(st["cache"][i][b, :, at], unit), st["cache"][i + 1][b, :, at]).masked_fill(~new[..., None, None], 0).to(torch.bfloat16)
            for i, unit in ((0, K_UNIT), (2, V_UNIT))]
    return [q] + back


def own_append(st, case):
    from ternainfer_b200.kv4 import kv4_append, kv4_read
    q = kv4_append(st["cache"], st["k"], st["v"], st["start"], st["counts"], q=st["q"], table=st["table"])
    return [q, *kv4_read(st["cache"], st["start"], case["tokens"], st["counts"])]


def plain_attend(st, case):
    B, T, H, K, D = (case[n] for n in ("batch", "tokens", "heads", "kv_heads", "dim"))
    kc, ks, vc, vs = st["cache"]
    L = case["past"] + T                                                # (what the longest sequence holds)
    k, v = values(unpack(kc[:, :, :L], K_UNIT), ks[:, :, :L]), values(unpack(vc[:, :, :L], V_UNIT), vs[:, :, :L])
    q = st["q"].float().view(B, T, K, H // K, D).permute(0, 2, 3, 1, 4).reshape(B, K, -1, D) / math.sqrt(D)
    score = (q @ k.transpose(-1, -2)).view(B, K, H // K, T, L)
    at = st["start"][:, None] + torch.arange(T, device=DEV)             # positions of the queries
    key = torch.arange(L, device=DEV)
    sees = key <= at[..., None]
    if case["window"]:
        sees &= key > at[..., None] - case["window"]
    score.masked_fill_(~sees[:, None, None], -math.inf)
    p = (score - score.amax(-1, keepdim=True)).exp()
    o = (p.view(B, K, -1, L) @ v) / p.sum(-1).view(B, K, -1, 1)
    return o.view(B, K, H // K, T, D).permute(0, 3, 1, 2, 4).reshape(B, T, H, D).to(torch.bfloat16)


def own_attend(st, case):
    from ternainfer_b200.kv4 import kv4_attend
    return kv4_attend(st["q"], st["cache"], st["start"], window=case["window"])


def plain_logprobs(st, case):
    x = st["logits"].float()
    m = x.amax(-1, keepdim=True)
    e = (x - m).exp()
    total = e.sum(-1, keepdim=True)
    lse = m + total.log()
    lp = (x.gather(-1, st["targets"][:, None]) - lse)[:, 0]
    p = e / total
    h = -torch.where(p > 0, p * (x - lse), torch.zeros_like(p)).sum(-1)
    if case["grad"]:
        gl, gh = st["grad_logprob"][:, None], st["grad_entropy"][:, None]
        d = -gl * p - gh * p * torch.where(p > 0, x - lse + h[:, None], torch.zeros_like(p))
        d.scatter_add_(-1, st["targets"][:, None], gl)
        return [lp, h, d.to(st["logits"].dtype)]
    ids = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, : case["top"]]     # (equal logits: the lowest id first)
    return [lp, h, x.gather(-1, ids) - lse, ids] if case["top"] else [lp, h]


def own_logprobs(st, case):
    from ternainfer_b200.scores import token_logprobs
    r = token_logprobs(st["logits"], st["targets"], top=case["top"])
    if case["grad"]:
        d, = torch.autograd.grad((r.logprob, r.entropy), st["logits"], (st["grad_logprob"], st["grad_entropy"]))
        return [r.logprob.detach(), r.entropy.detach(), d]
    return [r.logprob, r.entropy, r.top_logprob, r.top_token] if case["top"] else [r.logprob, r.entropy]


# ---------------------------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    kind = case["kind"]
    size = {"bfloat16": 2, "float16": 2, "float32": 4}.get(case.get("dtype"), 2)
    if kind == "logprobs":
        n = case["rows"] * case["vocab"]
        if case["grad"]:       # the forward's reading; the backward's, and its writing
            return {"bytes": 3 * n * size + case["rows"] * 32, "flops": 12 * n}
        return {"bytes": n * size + case["rows"] * (16 + 12 * case["top"]), "flops": 5 * n}
    B, T, H, K, D = (case[n] for n in ("batch", "tokens", "heads", "kv_heads", "dim"))
    row = D // 2 + D // GROUP * 2                                       # bytes of a key or a value in the cache
    if kind == "rotate":
        n = B * T * (H + K) * D * (2 if case["grad"] else 1)
        return {"bytes": 2 * n * size + B * T * case["rotary"] * 4, "flops": 3 * n * case["rotary"] / D}
    if kind == "append":       # queries read and written, keys and values read, their rows written and read back as bf16
        share = 0.75 if case["padded"] else 1.0
        return {"bytes": B * T * (4 * H * D + 4 * D + share * 2 * K * (2 * D + 2 * row) + 4 * K * D), "flops": B * T * (3 * (H + K) + 12 * K) * D}
    past = case["past"] if B == 1 else 0.75 * case["past"]
    seen = [min(past + t + 1, case["window"] or math.inf) for t in range(T)]
    held = min(past + T, (case["window"] or math.inf) + T - 1)
    return {"bytes": B * (held * K * 2 * row + 4 * T * H * D), "flops": 4 * B * H * D * sum(seen)}


# ---------------------------------------------------------------------------------------------- the definitions, in 64 bits

def exact(case, seed):
    st = _plain_state(case, seed)
    kind = case["kind"]
    if kind == "logprobs":
        x, t = st["logits"].double(), st["targets"]
        logp = torch.log_softmax(x, -1)
        lp = logp[torch.arange(case["rows"], device=DEV), t]
        h = -torch.special.xlogy(logp.exp(), logp.exp()).sum(-1)
        if case["grad"]:
            p = logp.exp()
            one = torch.nn.functional.one_hot(t, case["vocab"]).double() if p.numel() < 1 << 27 else None
            if one is None:
                return None
            return [lp, h, st["grad_logprob"].double()[:, None] * (one - p) - st["grad_entropy"].double()[:, None] * p * (logp + h[:, None])]
        if not case["top"]:
            return [lp, h]
        return [lp, h, torch.topk(logp, case["top"], -1).values, None]
    B, T, H, K, D = (case[n] for n in ("batch", "tokens", "heads", "kv_heads", "dim"))

    def spun(x, pos, rotary, half, scaling, sign):
        # complex numbers: a pair (a, b) times exp(i angle)
        inv, factor = angles(rotary, scaling)
        w = torch.polar(torch.full((1,), factor, dtype=torch.float64, device=DEV), sign * pos.double()[..., None, None] * inv)
        y = x.double().clone()
        a, b = (slice(0, rotary // 2), slice(rotary // 2, rotary)) if half else (slice(0, rotary, 2), slice(1, rotary, 2))
        z = torch.complex(y[..., a].contiguous(), y[..., b].contiguous()) * w
        y[..., a], y[..., b] = z.real, z.imag
        return y

    if kind == "rotate":
        said = (st["positions"], case["rotary"], case["half"], case["scaling"])
        out = [spun(st["q"], *said, 1), spun(st["k"], *said, 1)]
        return out + [spun(st["gq"], *said, -1), spun(st["gk"], *said, -1)] if case["grad"] else out
    if kind == "append":
        pos = st["start"][:, None] + torch.arange(T, device=DEV)
        q, k = (spun(st[n], pos, D, False, "none", 1) for n in "qk")
        gone = torch.zeros((B, T), dtype=torch.bool, device=DEV) if st["counts"] is None else torch.arange(T, device=DEV) >= st["counts"][:, None]

        def held(x):           # the nearest of the group's sixteen levels, the even one of two
            x = x.double().reshape(B, T, K, D // GROUP, GROUP)
            big = x.abs().amax(-1, keepdim=True)
            step = (torch.where((x == big).any(-1, keepdim=True), big, -big) / -8).half().double()
            near = torch.where(step == 0, 0.0, torch.clamp(torch.round(x / step), -8, 7) * step)
            return near.reshape(B, T, K, D).masked_fill(gone[..., None, None], 0)

        return [q, held(k.to(torch.bfloat16)), held(st["v"])]
    # attend
    kc, ks, vc, vs = st["cache"]
    out = torch.empty((B, T, H, D), dtype=torch.float64, device=DEV)
    for b in range(B):
        first = int(st["start"][b])
        n = first + T
        for h in range(K):
            k = (unpack(kc[b, h, :n], K_UNIT).double() - 8) * ks[b, h, :n].double().repeat_interleave(GROUP, -1)
            v = (unpack(vc[b, h, :n], V_UNIT).double() - 8) * vs[b, h, :n].double().repeat_interleave(GROUP, -1)
            ahead = torch.arange(n, device=DEV) - (first + torch.arange(T, device=DEV))[:, None]
            hidden = (ahead > 0) | (ahead <= -case["window"]) if case["window"] else ahead > 0
            for i in range(h * (H // K), (h + 1) * (H // K)):
                a = (st["q"][b, :, i].double() @ k.T / D ** 0.5).masked_fill_(hidden, -math.inf)
                out[b, :, i] = torch.softmax(a, -1) @ v
    return out


def _plain_state(case, seed):
    global own
    was, own = own, False
    try:
        return prepare(case, seed)
    finally:
        own = was
