"""The operators between a decoder layer's projections and its MoE FFN whose speed matters to a user of this library, as plain torch and as
the library's own calls: rotary positions (Context.rope), a cache that is quantised as it is written and read back (KvCache.write, read),
and attention over it for a batch that may share a prefix (KvCache.attend).  `kind`:
  rope    rotates the query and key heads of a fused projection's output, where they lie
  cache   writes `write` new rows of keys and values, then reads `read` rows back, the new ones last
  attend  one call for a batch of sequences, each with keys of its own behind a prefix that all of them share
"""
import math

import torch

own = False

DEV = torch.device("cuda", 0)
DTYPE = {"bf16": torch.bfloat16, "f32": torch.float32}
VALUE_BYTES = {"bf16": 2.0, "q8": 1.0, "q4": 0.5}

_ROPE = dict(kind="rope", heads=36, head_dim=128, n_rot=128, sections="64", interleaved=False, adjacent=False, inverse=False, x="bf16", base=1e6)
_CACHE = dict(kind="cache", cache="q8", n_kv=4, head_dim=128, page=64, x="bf16", out="bf16", padded=False)
_ATTEND = dict(kind="attend", cache="q8", n_head=32, n_kv=4, head_dim=128, page=64, x="bf16", new=1, prefix=0)


def listed():
    return [
        # the 32 query and 4 key heads of one token, one step of one sequence
        dict(_ROPE, name="rope_token", tokens=1),
        # a prompt with pictures in it: time, height and width take turns over the pairs
        dict(_ROPE, name="rope_pictures", tokens=2305, sections="24,20,20", interleaved=True),
        # the way back through half-rotated heads of adjacent pairs with two axes
        dict(_ROPE, name="rope_back", tokens=777, heads=20, n_rot=64, sections="16,16", adjacent=True, inverse=True, x="f32"),
        # a step of 64 sequences: a row each, written to pages all over the cache and read back
        dict(_CACHE, name="cache_step", write=64, read=64),
        # a prompt's chunk arrives, and the sequence is read back whole; the chunk is padded
        dict(_CACHE, name="cache_chunk", write=1000, read=5003, padded=True),
        # long prompts into the smallest cache, fp32 on either side
        dict(_CACHE, name="cache_prompts", cache="q4", write=16384, read=16384, n_kv=8, page=16, x="f32", out="f32"),
        # one sequence with a context of 4096 in an unquantised cache
        dict(_ATTEND, name="attend_one", cache="bf16", seqs=1, own_min=4096, own_max=4096),
        # a batch of ragged sequences
        dict(_ATTEND, name="attend_batch", seqs=64, own_min=200, own_max=4096),
        # the same instructions in front of every sequence
        dict(_ATTEND, name="attend_prefix", seqs=64, own_min=5, own_max=512, prefix=8192),
        # one long document in the smallest cache
        dict(_ATTEND, name="attend_document", cache="q4", seqs=1, own_min=131072, own_max=131072),
        # chunks of three prompts behind a shared prefix
        dict(_ATTEND, name="attend_chunks", seqs=3, own_min=197, own_max=1500, new=197, prefix=1000),
        # few short sequences in fp32, two query heads to a key head
        dict(_ATTEND, name="attend_short", cache="bf16", seqs=17, own_min=1, own_max=777, n_head=16, n_kv=8, head_dim=64, page=16, x="f32"),
    ]


def _between(rng, low, high):
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return v | 1 if v > 8 and rng.random() < 0.6 else v


def _cost(c):
    w = work(c)
    return max(w["bytes"] / 6.5e12, w["flops"] / 4e14)


def _held(c):
    """About the bytes that the plain form of an attention case holds at once."""
    tokens, keys = c["seqs"] * c["new"], c["prefix"] + c["own_max"]
    return 12.0 * tokens * c["n_head"] * keys + 16.0 * (c["seqs"] * c["own_max"] + c["prefix"]) * c["n_kv"] * c["head_dim"]


def draw(rng):
    kind = rng.choice(("rope", "cache", "attend", "attend"))
    most = max(_cost(c) for c in listed() if c["kind"] == kind)
    while True:
        if kind == "rope":
            head_dim = rng.choice((64, 128, 256))
            n_rot = rng.choice((head_dim, head_dim, head_dim // 2))
            axes = rng.choice((1, 1, 2, 3, 4))
            rest = [rng.randint(n_rot // 2 // (2 * axes), n_rot // 2 // axes) for _ in range(axes - 1)]
            c = dict(kind=kind, tokens=_between(rng, 1, 4096), heads=rng.choice((1, 5, 8, 18, 20, 36, 40)), head_dim=head_dim, n_rot=n_rot,
                     sections=",".join(str(s) for s in [n_rot // 2 - sum(rest)] + rest), interleaved=axes > 1 and rng.random() < 0.5,
                     adjacent=rng.random() < 0.4, inverse=rng.random() < 0.3, x=rng.choice(("bf16", "f32")), base=rng.choice((1e4, 5e5, 1e6)))
        elif kind == "cache":
            write = _between(rng, 1, 16384)
            c = dict(kind=kind, cache=rng.choice(("bf16", "q8", "q8", "q4", "q4")), n_kv=rng.choice((1, 2, 4, 5, 8)), head_dim=rng.choice((64, 128, 256)),
                     page=rng.choice((16, 32, 64, 128, 256)), x=rng.choice(("bf16", "f32")), out=rng.choice(("bf16", "f32")), write=write,
                     read=write + rng.choice((0, _between(rng, 1, 8192))), padded=rng.random() < 0.3)
        else:
            n_kv = rng.choice((1, 2, 4, 8))
            new = rng.choice((1, 1, 1, _between(rng, 2, 256)))
            own_max = max(new, _between(rng, 1, 131072))
            c = dict(kind=kind, cache=rng.choice(("bf16", "q8", "q8", "q4")), n_head=n_kv * rng.choice((1, 2, 3, 4, 7, 8, 16)), n_kv=n_kv,
                     head_dim=rng.choice((64, 128, 128, 256)), page=rng.choice((16, 32, 64, 128, 256)), x=rng.choice(("bf16", "bf16", "f32")), new=new,
                     prefix=rng.choice((0, _between(rng, 1, 16384))), seqs=_between(rng, 1, 128), own_min=max(new, own_max // rng.choice((1, 2, 8))), own_max=own_max)
            if _held(c) > 6e9:
                continue
        if _cost(c) <= most:
            return c


# ---- inputs ------------------------------------------------------------------------------------------------------------

def _rows(gen, n, heads, dim, dtype):
    """Keys or values: normal, with a few channels of every head that are larger than the others."""
    loud = 1.0 + 5.0 * (torch.rand((heads, dim), generator=gen, device=DEV) < 0.02)
    return (torch.randn((n, heads, dim), generator=gen, device=DEV) * loud).to(dtype)


def _grid(gen, tokens, axes):
    """Positions [axes][tokens]: a sequence that begins anywhere; with several axes text runs, pictures of 16 by 24 and text again."""
    start = int(torch.randint(0, 1 << 20, (1,), generator=gen, device=DEV))
    at = torch.arange(tokens, device=DEV)
    pos = (start + at).expand(axes, tokens).clone()
    if axes > 1:
        inside = (at % 512) >= 128
        cell = at % 512 - 128
        pos[0] = torch.where(inside, start + at // 512, pos[0])
        pos[1] = torch.where(inside, start + cell // 24, pos[1])
        for a in range(2, axes):
            pos[a] = torch.where(inside, start + cell % 24 + (a - 2), pos[a])
    return pos.to(torch.int32)


def _lengths(gen, c):
    """Own keys of each sequence, spread evenly between the case's bounds, in an order from the seed."""
    n = c["seqs"]
    even = [c["own_min"] + (c["own_max"] - c["own_min"]) * i // max(n - 1, 1) for i in range(n - 1)] + [c["own_max"]]
    return torch.tensor(even, dtype=torch.int32, device=DEV)[torch.randperm(n, generator=gen, device=DEV)]


def _new_tokens(c):
    """New tokens of each sequence: half to all of the case's `new`."""
    return [max(1, c["new"] - (c["new"] // 2) * i // max(c["seqs"] - 1, 1)) for i in range(c["seqs"])]


def _inputs(c, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    dt = DTYPE[c["x"]]
    if c["kind"] == "rope":
        sections = [int(s) for s in c["sections"].split(",")]
        qkv = torch.randn((c["tokens"], c["heads"] + 4, c["head_dim"]), generator=gen, device=DEV).to(dt)
        return {"x": qkv[:, :c["heads"]], "pos": _grid(gen, c["tokens"], len(sections)), "sections": sections}
    if c["kind"] == "cache":
        n_pages = -(-c["read"] // c["page"]) + 3
        slots = torch.randperm(n_pages, generator=gen, device=DEV)[:, None] * c["page"] + torch.arange(c["page"], device=DEV)
        slots = slots.reshape(-1)[:c["read"]].to(torch.int32)
        old = c["read"] - c["write"]
        s = {"n_pages": n_pages, "read_slots": slots, "write_slots": slots[old:].clone(),
             "k": _rows(gen, c["write"], c["n_kv"], c["head_dim"], dt), "v": _rows(gen, c["write"], c["n_kv"], c["head_dim"], dt),
             "old_slots": slots[:old], "old_k": _rows(gen, old, c["n_kv"], c["head_dim"], dt), "old_v": _rows(gen, old, c["n_kv"], c["head_dim"], dt)}
        if c["padded"]:    # rows that belong to nobody, behind the last token
            s["write_slots"] = torch.cat([s["write_slots"], torch.full((24,), -1, dtype=torch.int32, device=DEV)])
            s["k"], s["v"] = (torch.cat([s[n], _rows(gen, 24, c["n_kv"], c["head_dim"], dt)]) for n in ("k", "v"))
        return s
    new = _new_tokens(c)
    lens = _lengths(gen, c)
    per_seq, per_prefix = -(-c["own_max"] // c["page"]), -(-c["prefix"] // c["page"])
    n_pages = c["seqs"] * per_seq + per_prefix + 1
    order = torch.randperm(n_pages, generator=gen, device=DEV).to(torch.int32)
    rows = n_pages * c["page"]
    return {"n_pages": n_pages, "lens": lens, "pages": order[:c["seqs"] * per_seq].reshape(c["seqs"], per_seq),
            "prefix_pages": order[c["seqs"] * per_seq:c["seqs"] * per_seq + per_prefix],
            "q_start": torch.tensor([0] + [sum(new[:i + 1]) for i in range(len(new))], dtype=torch.int32, device=DEV), "new": new,
            "q": torch.randn((sum(new), c["n_head"], c["head_dim"]), generator=gen, device=DEV).to(dt),
            "k": _rows(gen, rows, c["n_kv"], c["head_dim"], torch.bfloat16), "v": _rows(gen, rows, c["n_kv"], c["head_dim"], torch.bfloat16)}


def prepare(case, seed):
    c = case
    s = _inputs(c, seed)
    s["case"] = c
    if own:
        from edge0_b200 import moe
        from edge0_b200.kv_cache import KvCache
        s["ctx"] = moe.Context(0)
    if c["kind"] == "rope":
        return s
    rows = s["n_pages"] * c["page"]
    if own:
        s["cache"] = KvCache(s["ctx"], kind=c["cache"], n_pages=s["n_pages"], page_size=c["page"], n_head_kv=c["n_kv"], head_dim=c["head_dim"])
        if c["kind"] == "cache":
            s["cache"].write(s["old_k"], s["old_v"], s["old_slots"])
        else:
            s["cache"].write(s.pop("k"), s.pop("v"), torch.arange(rows, dtype=torch.int32, device=DEV))
        return s
    for n in ("k", "v"):
        if c["kind"] == "cache":
            held = _quantised(torch.zeros((rows,) + s[n].shape[1:], device=DEV), c["cache"])
            for h, t in zip(held, _quantised(s["old_" + n], c["cache"])):
                h[s["old_slots"].long()] = t
        else:
            held = _quantised(s.pop(n), c["cache"])
        s["held_" + n] = held
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------------

def _quantised(x, cache):
    """What a cache holds of rows x: (values,) for bf16, else (codes, scales), a scale for a row (q8) or for 32 values (q4)."""
    if cache == "bf16":
        return (x.to(torch.bfloat16),)
    group, top = (x.shape[-1], 127) if cache == "q8" else (32, 7)
    g = x.double().reshape(x.shape[:-1] + (x.shape[-1] // group, group))
    d = (g.abs().amax(-1, keepdim=True) / top).float()
    d = d if cache == "q8" else d.to(torch.bfloat16).float()
    # the quotient in 64 bits: in 32 it lands on the border between two codes now and then
    code = torch.where(d > 0, g / d.double(), torch.zeros_like(g)).round().clamp(-top, top).to(torch.int8)
    return code.reshape(x.shape), d.squeeze(-1)


def _values(held, at):
    """The values that rows `at` of a cache stand for, in fp32."""
    if len(held) == 1:
        return held[0][at].float()
    code, d = held[0][at], held[1][at]
    return (code.float().reshape(d.shape + (code.shape[-1] // d.shape[-1],)) * d[..., None]).reshape(code.shape)


def _rope(s):
    c, x = s["case"], s["x"]
    half = c["n_rot"] // 2
    pair = torch.arange(half, device=DEV)
    sections = torch.tensor(s["sections"], device=DEV)
    axes = len(s["sections"])
    if c["interleaved"]:
        axis = torch.where(pair < axes * sections[pair % axes], pair % axes, 0)
    else:
        axis = (pair[:, None] >= sections.cumsum(0)).sum(-1)
    angle = s["pos"].double()[axis].T * c["base"] ** (-2.0 * pair.double() / c["n_rot"])
    cos, sin = angle.cos().float()[:, None], (-angle if c["inverse"] else angle).sin().float()[:, None]
    f = x.float()
    a, b = (f[..., 0:c["n_rot"]:2], f[..., 1:c["n_rot"]:2]) if c["adjacent"] else (f[..., :half], f[..., half:c["n_rot"]])
    turned = (a * cos - b * sin, a * sin + b * cos)
    turned = torch.stack(turned, dim=-1).flatten(-2) if c["adjacent"] else torch.cat(turned, dim=-1)
    return torch.cat([turned, f[..., c["n_rot"]:]], dim=-1).to(x.dtype)


def _cache(s):
    c = s["case"]
    n = c["write"]    # what is padded has no slot
    at, back = s["write_slots"][:n].long(), s["read_slots"].long()
    for held, new in ((s["held_k"], s["k"]), (s["held_v"], s["v"])):
        for h, t in zip(held, _quantised(new[:n], c["cache"])):
            h.index_copy_(0, at, t)
    return tuple(_values(held, back).to(DTYPE[c["out"]]) for held in (s["held_k"], s["held_v"]))


def _attend(s):
    c, q = s["case"], s["q"]
    T, B, Hk, G, D, M, P = q.shape[0], c["seqs"], c["n_kv"], c["n_head"] // c["n_kv"], c["head_dim"], c["new"], c["prefix"]
    token = torch.arange(T, device=DEV)
    seq = (token[:, None] >= s["q_start"][1:]).sum(-1)
    nth = token - s["q_start"].long()[seq]
    key = torch.arange(c["own_max"], device=DEV)
    at = s["pages"].long()[:, key // c["page"]] * c["page"] + key % c["page"]                                     # [B, own]
    front = torch.arange(P, device=DEV)
    front = s["prefix_pages"].long()[front // c["page"]] * c["page"] + front % c["page"]

    def padded(t):      # [T, Hk, G, n] -> [B, Hk, M * G, n], the tokens of a sequence together
        by_seq = torch.zeros((B, M) + t.shape[1:], device=DEV)
        by_seq[seq, nth] = t
        return by_seq.permute(0, 2, 1, 3, 4).reshape(B, Hk, M * G, t.shape[-1])

    def tokens(t):      # and back
        return t.reshape(B, Hk, M, G, t.shape[-1]).permute(0, 2, 1, 3, 4)[seq, nth]

    def heads_first(t):
        return t.permute(1, 0, 2, 3).reshape(Hk, T * G, t.shape[-1])

    f = q.float().reshape(T, Hk, G, D) / math.sqrt(D)
    mine = tokens(torch.matmul(padded(f), _values(s["held_k"], at).permute(0, 2, 3, 1)))                            # [T, Hk, G, own]
    seen = s["lens"].long()[seq] - (s["q_start"][1:] - s["q_start"][:-1]).long()[seq] + nth + 1
    mine = mine.masked_fill((key >= seen[:, None])[:, None, None], -math.inf)
    shared = torch.matmul(heads_first(f), _values(s["held_k"], front).permute(1, 2, 0)).reshape(Hk, T, G, P).transpose(0, 1)
    p = torch.cat([shared, mine], dim=-1)
    p = (p - p.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    out = torch.matmul(heads_first(p[..., :P]), _values(s["held_v"], front).transpose(0, 1)).reshape(Hk, T, G, D).transpose(0, 1)
    out = out + tokens(torch.matmul(padded(p[..., P:]), _values(s["held_v"], at).transpose(1, 2)))
    return out.reshape(q.shape).to(q.dtype)


def run(state):
    s = state
    c = s["case"]
    if not own:
        return {"rope": _rope, "cache": _cache, "attend": _attend}[c["kind"]](s)
    if c["kind"] == "rope":
        return s["ctx"].rope(s["x"], s["pos"], base=c["base"], n_rot=c["n_rot"], sections=s["sections"], interleaved=c["interleaved"],
                             adjacent=c["adjacent"], inverse=c["inverse"])
    if c["kind"] == "cache":
        s["cache"].write(s["k"], s["v"], s["write_slots"])
        return s["cache"].read(s["read_slots"], dtype=DTYPE[c["out"]])
    return s["cache"].attend(s["q"], s["lens"], s["pages"], max_kv_len=c["own_max"], q_start=None if c["new"] == 1 else s["q_start"], max_new=c["new"],
                             prefix_pages=s["prefix_pages"], prefix_len=c["prefix"])


def work(case):
    c = case
    if c["kind"] == "rope":
        n = c["tokens"] * c["heads"]
        axes = c["sections"].count(",") + 1
        return {"bytes": 2.0 * n * c["head_dim"] * (2 if c["x"] == "bf16" else 4) + 4.0 * axes * c["tokens"], "flops": 3.0 * n * c["n_rot"]}
    scales = {"bf16": 0, "q8": 4, "q4": 2 * c["head_dim"] // 32}[c["cache"]]
    row = 2 * c["n_kv"] * (c["head_dim"] * VALUE_BYTES[c["cache"]] + scales)     # a position's keys and values in the cache
    if c["kind"] == "cache":
        values = 2 * c["n_kv"] * c["head_dim"]
        size = {"bf16": 2, "f32": 4}
        return {"bytes": c["write"] * (values * size[c["x"]] + row) + c["read"] * (values * size[c["out"]] + row) + 4.0 * (c["write"] + c["read"]),
                "flops": 4.0 * values * c["write"] + values * c["read"]}
    new, n = _new_tokens(c), c["seqs"]
    mean = sum(c["own_min"] + (c["own_max"] - c["own_min"]) * i // max(n - 1, 1) for i in range(n - 1)) + c["own_max"]
    seen = sum(t * (mean / n + c["prefix"]) - t * (t - 1) / 2 for t in new)      # keys of all tokens, lengths at their mean
    return {"bytes": (mean + c["prefix"]) * row + 2.0 * sum(new) * c["n_head"] * c["head_dim"] * (2 if c["x"] == "bf16" else 4),
            "flops": 4.0 * c["n_head"] * c["head_dim"] * seen}


# ---- the definitions, in 64 bits -----------------------------------------------------------------------------------------

def _stored(x, cache):
    """The values that a cache stands for after rows x were written."""
    if cache == "bf16":
        return x.to(torch.bfloat16).double()
    n, top = (x.shape[-1], 127.0) if cache == "q8" else (32, 7.0)
    w = x.double().unflatten(-1, (-1, n))
    step = (w.abs().max(dim=-1).values / top).to(torch.float32)
    if cache == "q4":
        step = step.to(torch.bfloat16)
    step = step.double().unsqueeze(-1)
    return (torch.round(w / step.clamp(min=1e-300)).clamp(-top, top) * step).flatten(-2)


def exact(case, seed):
    c = case
    s = _inputs(c, seed)
    if c["kind"] == "rope":
        x, half = s["x"].double(), c["n_rot"] // 2
        out = x.clone()
        owner = [a for a, n in enumerate(s["sections"]) for _ in range(n)]
        if c["interleaved"]:
            A = len(s["sections"])
            owner = [i % A if i < A * s["sections"][i % A] else 0 for i in range(half)]
        for i in range(half):
            w = s["pos"][owner[i]].double() * math.pow(c["base"], -2.0 * i / c["n_rot"]) * (-1.0 if c["inverse"] else 1.0)
            z = torch.polar(torch.ones_like(w), w)[:, None]
            a, b = (2 * i, 2 * i + 1) if c["adjacent"] else (i, i + half)
            z = torch.complex(x[..., a], x[..., b]) * z
            out[..., a], out[..., b] = z.real, z.imag
        return out
    if c["kind"] == "cache":
        n = c["write"]
        return tuple(torch.cat([_stored(s["old_" + m], c["cache"]), _stored(s[m][:n], c["cache"])]) for m in ("k", "v"))
    D, G = c["head_dim"], c["n_head"] // c["n_kv"]
    held = lambda m, pages, n: _stored(s[m].reshape(-1, c["page"], c["n_kv"], D)[pages.long()].flatten(0, 1)[:n], c["cache"]).repeat_interleave(G, 1)  # noqa: E731
    front = [held(m, s["prefix_pages"], c["prefix"]) for m in ("k", "v")]
    out, t = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV), 0
    for b, (n, length) in enumerate(zip(s["new"], s["lens"].tolist())):
        k, v = (torch.cat([front[i], held(m, s["pages"][b], length)]) for i, m in enumerate(("k", "v")))
        score = torch.einsum("thd,khd->thk", s["q"][t:t + n].double(), k) / math.sqrt(D)
        last = c["prefix"] + length - n + torch.arange(n, device=DEV)
        score[(torch.arange(k.shape[0], device=DEV) > last[:, None])[:, None].expand_as(score)] = -math.inf
        out[t:t + n] = torch.einsum("thk,khd->thd", torch.softmax(score, dim=-1), v)
        t += n
    return out
