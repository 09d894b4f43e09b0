"""The operators around the attention half of a decoder block, as cases that can be timed one by one: low-rank adapters of
many requests beside a shared projection, norms and rotation of queries and keys on the rows that the merged projection wrote
(with and without the store into a paged cache), and attention of new tokens over that cache.  Shapes are those of the
benchmark's decoder (hidden 5120, 40 / 8 heads of 128, intermediate 17408) and of the served checkpoint's attention blocks
(24 / 4 heads of 256, gated output, a quarter of the head rotated); inputs are made on the GPU from the seed.

    listed()            the cases, each a dict of plain values with a name
    draw(rng)           one more case of the same ranges
    prepare(case, seed) what a program holds before the call
    run(state)          one pass: the plain form in 32 bits, or (own) the framework's operator
    exact(case, seed)   the operator's definition in 64 bits on the same inputs
    work(case)          bytes and flops the pass cannot do without
"""
import math
import random

import torch

own = False

HIDDEN, INTER = 5120, 17408
# rows of the shards and K of the layers an adapter stands beside
LAYERS = {"qkv": ((5120, 1024, 1024), HIDDEN), "o": ((HIDDEN,), 5120), "gate_up": ((INTER, INTER), HIDDEN), "down": ((HIDDEN,), INTER)}
# query heads, key-value heads, head size, rotated part, gated output
HEADS = {"plain": (40, 8, 128, 128, False), "gated": (24, 4, 256, 64, True)}


def listed():
    return [
        # one request with an adapter beside the merged qkv projection, one token: latency
        dict(name="adapters_qkv_m1", kind="adapters", layer="qkv", rank=16, bank=4, requests=1, tokens=1, spread=0),
        # nine requests of three tokens each, eight adapters in the bank, beside gate_up: a speculative step
        dict(name="adapters_gate_up_m27", kind="adapters", layer="gate_up", rank=32, bank=8, requests=9, tokens=3, spread=1),
        # sixty-four sequences in decode, some without an adapter, beside down
        dict(name="adapters_down_m64", kind="adapters", layer="down", rank=64, bank=16, requests=64, tokens=1, spread=2),
        # chunks of five prompts of different lengths in one batch
        dict(name="adapters_gate_up_m2051", kind="adapters", layer="gate_up", rank=16, bank=8, requests=5, tokens=0, total=2051, spread=3),
        # the decode step of eight sequences: norm, rotate, store into the cache
        dict(name="norm_rope_store_m8", kind="rope", heads="plain", tokens=8, store=True, interleaved=False, norm=True, scaling="none", far=40000, page=16),
        # a prompt chunk of the served checkpoint's attention block, stored
        dict(name="norm_rope_store_gated_m2051", kind="rope", heads="gated", tokens=2051, store=True, interleaved=False, norm=True, scaling="none", far=4096, page=16),
        # a long prompt at far positions, frequencies scaled, pairs side by side, no cache
        dict(name="norm_rope_m8192", kind="rope", heads="plain", tokens=8192, store=False, interleaved=True, norm=True, scaling="yarn", far=1000000, page=16),
        # one sequence of ordinary length: latency
        dict(name="attend_b1_517", kind="attend", heads="plain", batch=1, new=1, longest=517, ragged=False, page=16, head_major=True, spread=4),
        # eight sequences of different lengths in decode
        dict(name="attend_b8_8192", kind="attend", heads="plain", batch=8, new=1, longest=8192, ragged=True, page=16, head_major=True, spread=5),
        # the verification of four tokens of sixteen sequences, gated heads, a cache whose heads lie side by side
        dict(name="attend_gated_b16x4_16384", kind="attend", heads="gated", batch=16, new=4, longest=16384, ragged=True, page=16, head_major=False, spread=6),
        # one very long context
        dict(name="attend_b1_131072", kind="attend", heads="plain", batch=1, new=1, longest=131072, ragged=False, page=64, head_major=True, spread=7),
        # a full decode batch
        dict(name="attend_b64_16384", kind="attend", heads="plain", batch=64, new=1, longest=16384, ragged=True, page=16, head_major=True, spread=8),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(("adapters", "rope", "attend"))
    spread = rng.randrange(1 << 20)
    if kind == "adapters":
        case = dict(kind=kind, layer=rng.choice(sorted(LAYERS)), rank=rng.choice((8, 16, 16, 24, 32, 64, 128)), bank=_log_int(rng, 1, 16), spread=spread)
        if rng.random() < 0.5:       # decode or verification
            tokens = rng.randint(1, 4)
            return dict(case, requests=_log_int(rng, 1, 64 // tokens), tokens=tokens)
        return dict(case, requests=rng.randint(1, 8), tokens=0, total=_log_int(rng, 33, 2051))
    heads = rng.choice(sorted(HEADS))
    if kind == "rope":
        return dict(kind=kind, heads=heads, tokens=_log_int(rng, 1, 8192 if heads == "plain" else 4096), store=rng.random() < 0.6, interleaved=rng.random() < 0.3,
                    norm=rng.random() < 0.8, scaling=rng.choice(("none", "linear", "yarn")), far=_log_int(rng, 1000, 1000000), page=rng.choice((16, 16, 32, 64)))
    batch = _log_int(rng, 1, 96)
    return dict(kind=kind, heads=heads, batch=batch, new=rng.choice((1, 1, 1, 2, 3, 4)), longest=_log_int(rng, 64, min(131072, 262144 // batch)), ragged=rng.random() < 0.7,
                page=rng.choice((16, 16, 24, 32, 64)), head_major=rng.random() < 0.7, spread=spread)


# ---- what follows from a case alone ------------------------------------------------------------------------

def _row_ids(case):
    """The adapter of each row: the rows of a request stand together, one request in eight has no adapter."""
    rng = random.Random(case["spread"])
    sizes = [case["tokens"]] * case["requests"]
    if not case["tokens"]:
        cuts = sorted(rng.sample(range(1, case["total"]), case["requests"] - 1))
        sizes = [b - a for a, b in zip([0] + cuts, cuts + [case["total"]])]
    who = [i % case["bank"] if i == 0 else (-1 if rng.random() < 0.125 else rng.randrange(case["bank"])) for i in range(len(sizes))]
    return [w for w, n in zip(who, sizes) for _ in range(n)]


def _lens(case):
    """Keys of each sequence, those of its new tokens among them; a ragged batch holds a padding entry now and then."""
    rng = random.Random(case["spread"])
    longest, new = case["longest"], case["new"]
    if not case["ragged"]:
        return [longest] * case["batch"]
    some = [longest] + [max(new, int(longest * 16 ** -rng.random())) for _ in range(case["batch"] - 1)]
    return [0 if i and rng.random() < 0.04 else n for i, n in enumerate(some)]


def _frequencies(case, dims):
    """Radians per position of each rotated pair in 64 bits, and the factor on the rotated values: as they are, positions divided by
    eight, or the slow pairs divided by eight, the fast ones kept and a ramp between them."""
    inv = 1e6 ** (-torch.arange(0, dims, 2, dtype=torch.float64, device="cuda") / dims)
    if case["scaling"] == "none":
        return inv, 1.0
    if case["scaling"] == "linear":
        return inv / 8, 1.0
    turns = 32768 * inv / (2 * math.pi)                  # over the context the model was trained on
    at = lambda t: dims * math.log(32768 / (t * 2 * math.pi)) / (2 * math.log(1e6))  # noqa: E731  the pair that makes t turns
    lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), dims - 1)
    keep = 1 - ((torch.arange(turns.numel(), dtype=torch.float64, device="cuda") - lo) / max(hi - lo, 0.001)).clamp(0, 1)
    return inv / 8 * (1 - keep) + inv * keep, 0.1 * math.log(8) + 1


# ---- inputs ------------------------------------------------------------------------------------------------

def _normal(g, *shape, std=1.0):
    return (torch.randn(shape, device="cuda", generator=g) * std).to(torch.bfloat16)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(1000 * int(seed) + 17)
    kind = case["kind"]
    if kind == "adapters":
        rows, k = LAYERS[case["layer"]]
        ids = torch.tensor(_row_ids(case), dtype=torch.int32, device="cuda")
        m, n, r = ids.numel(), sum(rows), case["rank"]
        return {"kind": kind, "rows": list(rows), "ids": ids, "x": _normal(g, m, k), "base": _normal(g, m, n),
                "a": _normal(g, case["bank"], len(rows) * r, k, std=k ** -0.5), "b": _normal(g, case["bank"], n, r, std=r ** -0.5),
                "scales": 0.5 + torch.rand(case["bank"], len(rows), device="cuda", generator=g), "out": torch.empty(m, n, dtype=torch.bfloat16, device="cuda")}
    hq, hk, d, dims, gated = HEADS[case["heads"]]
    if kind == "rope":
        t, page = case["tokens"], case["page"]
        inv, amp = _frequencies(case, dims)
        state = {"kind": kind, "heads": case["heads"], "inv_freq": inv, "amplitude": amp, "interleaved": case["interleaved"],
                 "qkv": _normal(g, t, (2 if gated else 1) * hq * d + 2 * hk * d),
                 "positions": torch.randint(0, case["far"], (t,), device="cuda", generator=g),
                 "q_norm": 1 + _normal(g, d, std=0.1) if case["norm"] else None, "k_norm": 1 + _normal(g, d, std=0.1) if case["norm"] else None}
        if case["store"]:      # page 0 belongs to nobody; tokens go to slots of the others, in no order
            pages = -(-t // page) + 4
            slots = page + torch.randperm((pages - 1) * page, device="cuda", generator=g)[:t]
            state |= {"slots": torch.where(torch.rand(t, device="cuda", generator=g) < 0.03, -1, slots), "k_pages": _normal(g, pages, hk, page, d).transpose(1, 2),
                      "v_pages": _normal(g, pages, hk, page, d).transpose(1, 2)}
        return state
    lens, page, new = _lens(case), case["page"], case["new"]
    width = -(-max(lens) // page)
    pages = sum(-(-n // page) for n in lens) + 3
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    first, table = 0, torch.zeros(len(lens), width, dtype=torch.int32, device="cuda")
    for b, n in enumerate(lens):
        used = -(-n // page)
        table[b, :used] = order[first:first + used]
        first += used
    cache = [_normal(g, pages, hk, page, d).transpose(1, 2) if case["head_major"] else _normal(g, pages, page, hk, d) for _ in range(2)]
    t = len(lens) * new
    state = {"kind": kind, "k_pages": cache[0], "v_pages": cache[1], "table": table, "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"),
             "q": _normal(g, t, hq, d, std=1.5), "gate": None}
    if gated:
        state["gate"] = _normal(g, t, hq, 2 * d)[..., d:]        # as the projection leaves it: behind each head's query
    return state


# ---- one pass ------------------------------------------------------------------------------------------------

def _adapters_plain(s):
    """All adapters' inner products, those of the rows' own kept, then all outer products."""
    bank, n, r = s["b"].shape
    shards = len(s["rows"])
    mine = torch.where(s["ids"][:, None] == torch.arange(bank, device="cuda"), 1.0, 0.0)[:, :, None] * s["scales"]
    inner = (s["x"].float() @ s["a"].float().reshape(bank * shards * r, -1).T).view(-1, bank, shards, r) * mine[..., None]
    parts = s["b"].float().split(s["rows"], dim=1)
    delta = [inner[:, :, j].reshape(-1, bank * r) @ p.transpose(1, 2).reshape(bank * r, -1) for j, p in enumerate(parts)]
    return (s["base"].float() + torch.cat(delta, dim=1)).to(torch.bfloat16)


def _norm(x, weight, eps=1e-6):
    x = x.float()
    return x if weight is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * weight.float()


def _turn(x, cos, sin, interleaved):
    dims = 2 * cos.shape[-1]
    one, two = (x[..., 0:dims:2], x[..., 1:dims:2]) if interleaved else (x[..., :dims // 2], x[..., dims // 2:dims])
    one, two = one * cos - two * sin, two * cos + one * sin
    turned = torch.stack((one, two), dim=-1).flatten(-2) if interleaved else torch.cat((one, two), dim=-1)
    return torch.cat((turned, x[..., dims:]), dim=-1)


def _heads_of(qkv, heads):
    hq, hk, d, _, gated = HEADS[heads]
    w = (2 if gated else 1) * d
    q, k, v = qkv.split((hq * w, hk * d, hk * d), dim=1)
    return q.unflatten(1, (hq, w))[..., :d], k.unflatten(1, (hk, d)), v.unflatten(1, (hk, d))


def _rope_plain(s):
    q, k, v = _heads_of(s["qkv"], s["heads"])
    angle = s["positions"].double()[:, None, None] * s["inv_freq"]                  # far positions: 64 bits
    cos, sin = (angle.cos() * s["amplitude"]).float(), (angle.sin() * s["amplitude"]).float()
    q = _turn(_norm(q, s["q_norm"]), cos, sin, s["interleaved"]).to(torch.bfloat16)
    k = _turn(_norm(k, s["k_norm"]), cos, sin, s["interleaved"]).to(torch.bfloat16)
    if "slots" not in s:
        return [q, k]
    page = s["k_pages"].shape[1]
    keep, at = (s["slots"] >= 0)[:, None, None], s["slots"].clamp(min=0)             # tokens without a slot write page 0's first row as it is
    where = (at // page, at % page)
    s["k_pages"][where] = torch.where(keep, k, s["k_pages"][where])
    s["v_pages"][where] = torch.where(keep, v, s["v_pages"][where])
    return [q, s["k_pages"], s["v_pages"]]


def _attend_plain(s):
    batch, width = s["table"].shape
    t, hq, d = s["q"].shape
    page, hk = s["k_pages"].shape[1:3]
    new = t // batch
    keys = s["k_pages"][s["table"]].reshape(batch, width * page, hk, d).permute(0, 2, 3, 1).float()
    values = s["v_pages"][s["table"]].reshape(batch, width * page, hk, d).transpose(1, 2).float()
    q = s["q"].view(batch, new, hk, hq // hk, d).transpose(1, 2).float()
    scores = (q.reshape(batch, hk, -1, d) @ keys).view(batch, hk, new, hq // hk, -1) * d ** -0.5
    last = s["lens"][:, None] - new + torch.arange(new, device="cuda")                 # the last key each token sees
    seen = (torch.arange(width * page, device="cuda") <= last[..., None])[:, None, :, None, :]
    top = scores.masked_fill(~seen, -math.inf).amax(-1, keepdim=True)
    p = torch.where(seen, torch.exp(scores - torch.where(top == -math.inf, 0.0, top)), 0.0)
    total = p.sum(-1, keepdim=True)
    o = (p.reshape(batch, hk, -1, p.shape[-1]) @ values).view(batch, hk, new, hq // hk, d) / torch.where(total == 0, 1.0, total)
    o = o.transpose(1, 2).reshape(t, hq, d)
    if s["gate"] is not None:
        o = o * torch.sigmoid(s["gate"].float())
    return o.to(torch.bfloat16)


def run(state):
    s = state
    if own:
        from hyperqwen_rtx4080s32_b200 import ops

        if s["kind"] == "adapters":
            return ops.low_rank_add(s["base"], s["x"], s["a"], s["b"], s["scales"], s["ids"], s["rows"], out=s["out"])
        if s["kind"] == "rope":
            hq, hk, d, _, gated = HEADS[s["heads"]]
            how = dict(q_norm=s["q_norm"], k_norm=s["k_norm"], eps=1e-6, amplitude=s["amplitude"], interleaved=s["interleaved"], gated=gated)
            if "slots" not in s:
                return list(ops.qk_norm_rope(s["qkv"], s["positions"], s["inv_freq"], hq, hk, d, **how))
            q = ops.qk_norm_rope_store(s["qkv"], s["positions"], s["inv_freq"], hq, hk, d, s["k_pages"], s["v_pages"], s["slots"], **how)
            return [q, s["k_pages"], s["v_pages"]]
        return ops.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], gate=s["gate"])
    if s["kind"] == "adapters":
        return _adapters_plain(s)
    if s["kind"] == "rope":
        return _rope_plain(s)
    return _attend_plain(s)


# ---- the definitions in 64 bits ----------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "adapters":
        out = s["base"].double()
        edges = [sum(s["rows"][:j]) for j in range(len(s["rows"]) + 1)]
        r = case["rank"]
        for who in sorted(set(_row_ids(case)) - {-1}):
            mine = (s["ids"] == who).nonzero()[:, 0]
            for j in range(len(s["rows"])):
                inner = s["x"][mine].double() @ s["a"][who, j * r:(j + 1) * r].double().T
                out[mine, edges[j]:edges[j + 1]] += float(s["scales"][who, j]) * (inner @ s["b"][who, edges[j]:edges[j + 1]].double().T)
        return out
    hq, hk, d, dims, gated = HEADS[case["heads"]]
    if case["kind"] == "rope":
        t, half = case["tokens"], dims // 2
        wide = (2 if gated else 1) * d
        at_q = torch.arange(hq, device="cuda")[:, None] * wide + torch.arange(d, device="cuda")
        at_k = hq * wide + torch.arange(hk * d, device="cuda").view(hk, d)
        p = torch.arange(half, device="cuda")
        i, j = (2 * p, 2 * p + 1) if case["interleaved"] else (p, p + half)
        turn = torch.polar(torch.full((t, 1, half), float(s["amplitude"]), dtype=torch.float64, device="cuda"),
                           s["positions"].double().view(t, 1, 1) * s["inv_freq"].double())
        found = []
        for at, weight in ((at_q, s["q_norm"]), (at_k, s["k_norm"])):
            u = s["qkv"][:, at].double()
            if weight is not None:
                u = u / (u.pow(2).sum(-1, keepdim=True) / d + 1e-6).sqrt() * weight.double()
            z = torch.complex(u[..., i], u[..., j]) * turn
            u[..., i], u[..., j] = z.real, z.imag
            found.append(u)
        if not case["store"]:
            return found
        k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
        kept = (s["slots"] >= 0).nonzero()[:, 0]
        page, row = s["slots"][kept].div(case["page"], rounding_mode="floor"), s["slots"][kept].remainder(case["page"])
        k_pages[page, row] = found[1][kept]
        v_pages[page, row] = s["qkv"][kept][:, hq * wide + hk * d:].double().view(-1, hk, d)
        return [found[0], k_pages, v_pages]
    new, page = case["new"], case["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lens(case)):
        at = torch.arange(n, device="cuda")
        pages, row = s["table"][b, at // page].long(), at % page
        for h in range(hk if n else 0):
            k, v = s["k_pages"][pages, row, h].double(), s["v_pages"][pages, row, h].double()
            for i in range(new):
                sees = n - new + i + 1
                if sees > 0:
                    mine = slice(h * (hq // hk), (h + 1) * (hq // hk))
                    w = torch.softmax(s["q"][b * new + i, mine].double() @ k[:sees].T / math.sqrt(d), dim=-1)
                    out[b * new + i, mine] = w @ v[:sees]
    if s["gate"] is not None:
        out /= 1 + torch.exp(-s["gate"].double())
    return out


# ---- what a pass cannot do without ---------------------------------------------------------------------------

def work(case):
    if case["kind"] == "adapters":
        rows, k = LAYERS[case["layer"]]
        ids, n, r = _row_ids(case), sum(rows), case["rank"]
        m, used, with_one = len(ids), len(set(ids) - {-1}), sum(i >= 0 for i in ids)
        return {"bytes": 2 * with_one * k + 4 * m * n + 2 * used * r * (len(rows) * k + n) + 4 * m, "flops": 2.0 * with_one * r * (len(rows) * k + n)}
    hq, hk, d, dims, gated = HEADS[case["heads"]]
    if case["kind"] == "rope":
        t = case["tokens"]
        return {"bytes": t * (4 * (hq + hk) * d + 8 + (4 * hk * d + 8 if case["store"] else 0)), "flops": 10.0 * t * (hq + hk) * d}
    lens, new = _lens(case), case["new"]
    keys, t = sum(lens), len(lens) * new
    seen = sum(max(0, n - new + i + 1) for n in lens for i in range(new))
    return {"bytes": 4 * keys * hk * d + t * hq * d * (6 if gated else 4) + 4 * sum(-(-n // case["page"]) for n in lens) + 4 * len(lens), "flops": 4.0 * seen * hq * d}
