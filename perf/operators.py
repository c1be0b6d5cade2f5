"""What is measured of the single-token serving operators: block tables and slot maps, the attention input side with
several rotary axes, attention of one new token over the paged cache, and linear attention with a decay for each head
(chunked for prompts, recurrent for single tokens).

The pages have the prefix pool's geometry: a page holds 32 tokens of keys and values of every attention layer,
kv[page][layer][K|V][token][head][dim] bf16, or a whole number of recurrent states, state[page][slot][128][128] fp32;
a row's block table lists its state pages, its convolution pages, then its key/value pages. Requests' lengths are
spread evenly between a case's bounds and dealt to the rows by the seed, so a case's work does not depend on it."""

import math

import torch

own = False

PAGE = 32                       # tokens of a key/value page
HEADS, KV_HEADS, DIM = 8, 2, 256   # attention heads of the served layout, their width
ROT = 64                        # rotated dimensions of a head
PROJ = HEADS * 2 * DIM + 2 * KV_HEADS * DIM   # query and gate interleaved per head, then keys, then values
FIXED = 50                      # state and convolution pages ahead of the key/value pages in a block table
LAYERS = 6                      # attention layers of a page
LIN_HEADS, LIN_DIM = 16, 128    # recurrent layers: heads, key and value width
LIN_LAYERS = 18
HEADS_PER_PAGE = 6              # recurrent states of a page
STATE_PAGES = LIN_LAYERS * LIN_HEADS // HEADS_PER_PAGE
THETA = 1e7
EPS = 1e-6


def listed():
    return [
        # every row of a full batch has one more token: the call before each step of 64 conversations
        {"name": "tables_step", "op": "tables", "rows": 64, "lo": 0, "hi": 8192, "new_lo": 1, "new_hi": 1,
         "tokens": 64, "fixed": False},
        # ragged new prompts packed into one pass of the largest size, each row taking its state pages too
        {"name": "tables_prompts", "op": "tables", "rows": 256, "lo": 0, "hi": 0, "new_lo": 1, "new_hi": 126,
         "tokens": 16384, "fixed": True},
        # one token a row, text and image positions, keys and values straight into the cache
        {"name": "prep_step", "op": "prep", "tokens": 64, "axes": 3, "interleaved": True, "paged": True,
         "reach": 8192},
        # a pass of prompts with images: keys and values for the pass's own attention
        {"name": "prep_pass", "op": "prep", "tokens": 16384, "axes": 3, "interleaved": False, "paged": False,
         "reach": 131072},
        # one conversation over a 1,000-token prefix: latency
        {"name": "decode_row", "op": "decode", "rows": 1, "lo": 1000, "hi": 1000, "heads": 8, "kv_heads": 2,
         "dim": 256, "layers": 6, "gated": True},
        # a full batch with mixed lengths up to the longest prefix
        {"name": "decode_ragged", "op": "decode", "rows": 64, "lo": 1, "hi": 8192, "heads": 8, "kv_heads": 2,
         "dim": 256, "layers": 6, "gated": True},
        # another head layout: narrower heads, more of them, no gate
        {"name": "decode_heads", "op": "decode", "rows": 33, "lo": 100, "hi": 4096, "heads": 32, "kv_heads": 8,
         "dim": 128, "layers": 2, "gated": False},
        # one prompt of odd length
        {"name": "scan_row", "op": "scan", "rows": 1, "tokens": 1001, "lo": 1001, "per_token": True},
        # a pass of 64 rows of 128 new tokens, padded, each from its own cached state
        {"name": "scan_pass", "op": "scan", "rows": 64, "tokens": 128, "lo": 32, "per_token": True},
        # two of the longest prompts, a constant decay for each head
        {"name": "scan_long", "op": "scan", "rows": 2, "tokens": 8192, "lo": 8192, "per_token": False},
        # one token of one conversation, and of a full batch with the delta rule's correction
        {"name": "step_row", "op": "step", "rows": 1, "delta": False, "per_token": True},
        {"name": "step_batch", "op": "step", "rows": 64, "delta": True, "per_token": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["tables", "prep", "decode", "scan", "step"])
    if op == "tables":
        rows, hi = _log(rng, 1, 1000), rng.choice([0, _log(rng, 1, 8192)])
        new = _log(rng, 1, 300)
        new = min(new, 2 * 16384 // rows - 1)
        return {"op": op, "rows": rows, "lo": 0, "hi": hi, "new_lo": rng.choice([0, 1]), "new_hi": max(1, new),
                "tokens": rng.choice([16384, rows * (max(1, new) + 1)]), "fixed": rng.random() < 0.5}
    if op == "prep":
        return {"op": op, "tokens": _log(rng, 1, 16384), "axes": rng.choice([1, 2, 3, 3, 4]),
                "interleaved": rng.random() < 0.5, "paged": rng.random() < 0.5, "reach": _log(rng, 1000, 1000000)}
    if op == "decode":
        heads, kv_heads, dim, layers, gated = rng.choice([(8, 2, 256, 6, True), (8, 2, 256, 6, False),
                                                          (32, 8, 128, 2, False), (16, 2, 128, 2, True),
                                                          (12, 12, 64, 2, False), (6, 2, 256, 1, True)])
        rows = _log(rng, 1, 64)
        hi = _log(rng, 1, 4096)
        return {"op": op, "rows": rows, "lo": rng.choice([1, hi, (hi + 1) // 2]), "hi": hi, "heads": heads,
                "kv_heads": kv_heads, "dim": dim, "layers": layers, "gated": gated}
    if op == "scan":
        tokens = _log(rng, 1, 8192)
        rows = _log(rng, 1, max(1, min(64, 16384 // tokens)))
        return {"op": op, "rows": rows, "tokens": tokens, "lo": rng.choice([tokens, (tokens + 1) // 2]),
                "per_token": rng.random() < 0.7}
    return {"op": op, "rows": _log(rng, 1, 64), "delta": rng.random() < 0.5, "per_token": rng.random() < 0.7}


# ---------------------------------------------------------------- inputs


def _spread(count, lo, hi):
    """`count` whole numbers spread evenly over [lo, hi], the ends among them."""
    if count == 1:
        return [hi]
    return [lo + (hi - lo) * i // (count - 1) for i in range(count)]


def _pages(tokens):
    return -(-tokens // PAGE)


def _sections(axes):
    return {1: (32,), 2: (16, 16), 3: (11, 11, 10), 4: (8, 8, 8, 8)}[axes]


def _axis_of(axes, interleaved):
    """The axis whose position turns each of the 32 frequencies."""
    sections = _sections(axes)
    if not interleaved:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    return [i % axes if i // axes < sections[i % axes] else 0 for i in range(sum(sections))]


def _dealt(values, gen):
    order = torch.randperm(len(values), generator=gen, device="cuda")
    return torch.tensor(values, dtype=torch.int32, device="cuda")[order]


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.bfloat16):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)

    state = {"case": case}
    if case["op"] == "tables":
        rows = case["rows"]
        lengths = _dealt(_spread(rows, case["lo"], case["hi"]), gen)
        new = _dealt(_spread(rows, case["new_lo"], case["new_hi"]), gen)
        width = FIXED + _pages(case["hi"] + case["new_hi"])
        count = rows * width + 2
        ids = (torch.randperm(count - 2, generator=gen, device="cuda") + 2).int()
        tables = torch.zeros(rows, width, dtype=torch.int32, device="cuda")
        held = torch.where((lengths > 0) | (not case["fixed"]), FIXED, 0) + (lengths + PAGE - 1) // PAGE
        have = torch.arange(width, device="cuda") < held[:, None]
        tables[have] = ids[:int(have.sum())]
        state |= {"lengths": lengths, "new": new, "tables": tables, "free": ids[int(have.sum()):].contiguous()}
    elif case["op"] == "prep":
        t = case["tokens"]
        state["pr"] = normal(t, PROJ)
        state["q_w1"] = 1 + 0.1 * normal(DIM, dtype=torch.float32)
        state["k_w1"] = 1 + 0.1 * normal(DIM, dtype=torch.float32)
        state["inv_freq"] = 1.0 / (THETA ** (torch.arange(0, ROT, 2, dtype=torch.float32, device="cuda") / ROT))
        state["positions"] = torch.randint(0, case["reach"], (case["axes"], t), generator=gen, device="cuda",
                                           dtype=torch.int32)
        state["axis_of"] = torch.tensor(_axis_of(case["axes"], case["interleaved"]), device="cuda")
        state["layer"] = seed % LAYERS
        if case["paged"]:
            count = _pages(2 * t) + 2
            state["kv"] = torch.zeros(count, LAYERS, 2, PAGE, KV_HEADS, DIM, dtype=torch.bfloat16, device="cuda")
            state["slots"] = torch.randperm((count - 2) * PAGE, generator=gen, device="cuda")[:t] + 2 * PAGE
    elif case["op"] == "decode":
        rows, layer = case["rows"], seed % case["layers"]
        lengths = _dealt(_spread(rows, case["lo"], case["hi"]), gen)
        held = (lengths + PAGE - 1) // PAGE
        have = torch.arange(_pages(case["hi"]), device="cuda") < held[:, None]
        used = sum(_pages(n) for n in _spread(rows, case["lo"], case["hi"]))
        kv = torch.zeros(used + 2, case["layers"], 2, PAGE, case["kv_heads"], case["dim"], dtype=torch.bfloat16,
                         device="cuda")
        kv[:, layer] = normal(used + 2, 2, PAGE, case["kv_heads"], case["dim"])
        tables = torch.zeros(rows, FIXED + have.shape[1], dtype=torch.int32, device="cuda")
        tables[:, :FIXED] = 1
        tables[:, FIXED:][have] = (torch.randperm(used, generator=gen, device="cuda") + 2).int()
        state |= {"lengths": lengths, "kv": kv, "tables": tables, "layer": layer,
                  "q": normal(rows, case["heads"], case["dim"])}
        if case["gated"]:
            state["pr"] = normal(rows, 2 * (case["heads"] + case["kv_heads"]) * case["dim"])
    else:
        rows, layer = case["rows"], seed % LIN_LAYERS
        places = (rows,) if case["op"] == "step" else (rows, case["tokens"])
        q, k = normal(*places, LIN_HEADS, LIN_DIM), normal(*places, LIN_HEADS, LIN_DIM)
        unit = [x.float() * torch.rsqrt(x.float().square().sum(-1, keepdim=True) + EPS) for x in (q, k)]
        # the decay of the served layers, -exp(A_log) softplus(a + dt_bias): a decay for each token, or each head's own
        a_neg = -(1 + 15 * torch.rand(LIN_HEADS, generator=gen, device="cuda"))
        dt = normal(*places, LIN_HEADS, dtype=torch.float32) - 4
        g = a_neg * torch.log1p(torch.exp(dt)) if case["per_token"] else a_neg * 0.004
        ids = torch.randperm(2 * rows * STATE_PAGES, generator=gen, device="cuda").int() + 2
        pages = torch.zeros(2 * rows * STATE_PAGES + 2, HEADS_PER_PAGE, LIN_DIM, LIN_DIM, device="cuda")
        tables = torch.ones(2, rows, FIXED, dtype=torch.int32, device="cuda")
        tables[:, :, :STATE_PAGES] = ids.view(2, rows, STATE_PAGES)
        page, slot = _state_at(tables[0], layer)
        pages[page, slot] = 0.3 * normal(rows, LIN_HEADS, LIN_DIM, LIN_DIM, dtype=torch.float32)
        state |= {"q": unit[0].bfloat16(), "k": unit[1].bfloat16(), "v": normal(*places, LIN_HEADS, LIN_DIM), "g": g,
                  "pages": pages, "tables": tables[0], "out_tables": tables[1], "layer": layer}
        if case["op"] == "scan":
            state["real"] = _dealt(_spread(rows, case["lo"], case["tokens"]), gen)
        elif case["delta"]:
            state["beta"] = torch.sigmoid(normal(rows, LIN_HEADS, dtype=torch.float32)).bfloat16()
    return state


def _state_at(tables, layer):
    """(page, slot) of every (row, head) of a recurrent layer."""
    flat = layer * LIN_HEADS + torch.arange(LIN_HEADS, device=tables.device)
    return tables[:, flat // HEADS_PER_PAGE].long(), (flat % HEADS_PER_PAGE).expand(tables.shape[0], -1)


# ---------------------------------------------------------------- one pass


def run(state):
    return {"tables": _tables, "prep": _prep, "decode": _decode, "scan": _scan, "step": _step}[state["case"]["op"]](state)


def _tables(s):
    case = s["case"]
    if own:
        from jeff_b200 import kernels

        m = kernels.block_tables(s["lengths"], s["new"], s["free"], s["tables"], FIXED, case["tokens"],
                                 fixed=case["fixed"])
        return {"tables": s["tables"], "slots": m.slots, "rows": m.rows, "positions": m.positions,
                "starts": m.starts, "taken": m.taken}
    lengths, new, free, tables, tokens = s["lengths"].long(), s["new"].long(), s["free"], s["tables"], case["tokens"]
    held, need = (lengths + PAGE - 1) // PAGE, (lengths + new + PAGE - 1) // PAGE
    fresh = (lengths == 0) & (new > 0) if case["fixed"] else torch.zeros_like(lengths, dtype=torch.bool)
    take = torch.where(fresh, FIXED, 0) + need - held
    starts = torch.nn.functional.pad(new.cumsum(0), (1, 0))
    taken = torch.nn.functional.pad(take.cumsum(0), (1, 0))
    first = torch.where(fresh, 0, FIXED + held)
    entry = torch.arange(tables.shape[1], device=tables.device)
    at = taken[:-1, None] + entry - first[:, None]
    fill = (entry >= first[:, None]) & (entry < first[:, None] + take[:, None])
    got = torch.where(at < len(free), free[at.clamp(0, len(free) - 1)], 0)
    tables.copy_(torch.where(fill, got, tables))
    t = torch.arange(tokens, device=tables.device)
    row = torch.searchsorted(starts[1:], t, right=True)
    live = t < starts[-1]
    row = row.clamp(max=len(new) - 1)
    pos = lengths[row] + t - starts[row]
    page = tables[row, (FIXED + pos // PAGE).clamp(max=tables.shape[1] - 1)].long()
    return {"tables": tables, "slots": torch.where(live, page * PAGE + pos % PAGE, -1),
            "rows": torch.where(live, row, -1).int(), "positions": torch.where(live, pos, 0).int(),
            "starts": starts.int(), "taken": taken.int()}


def _prep(s):
    case, t = s["case"], s["case"]["tokens"]
    if own:
        from jeff_b200 import kernels

        axes = kernels.rope_axes(_sections(case["axes"]), case["interleaved"])
        if case["paged"]:
            q = kernels.attn_prep_axes(s["pr"], s["q_w1"], s["k_w1"], s["inv_freq"], s["positions"], axes,
                                       kv=s["kv"], attn_layer=s["layer"], slots=s["slots"])
            return {"q": q, "kv": s["kv"]}
        kn, vn = (torch.empty(t, KV_HEADS, DIM, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        q = kernels.attn_prep_axes(s["pr"], s["q_w1"], s["k_w1"], s["inv_freq"], s["positions"], axes, kn=kn, vn=vn)
        return {"q": q, "kn": kn, "vn": vn}
    pr = s["pr"]
    q = pr[:, :HEADS * 2 * DIM].view(t, HEADS, 2 * DIM)[:, :, :DIM].float()
    k = pr[:, HEADS * 2 * DIM:HEADS * 2 * DIM + KV_HEADS * DIM].view(t, KV_HEADS, DIM).float()
    v = pr[:, HEADS * 2 * DIM + KV_HEADS * DIM:].view(t, KV_HEADS, DIM)
    angle = s["positions"][s["axis_of"]].T.double() * s["inv_freq"].double()   # (t, 32); far positions need 64 bits
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turn(x, w1):
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w1
        a, b = x[..., :ROT // 2], x[..., ROT // 2:ROT]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., ROT:]], -1).bfloat16()

    q, k = turn(q, s["q_w1"]), turn(k, s["k_w1"])
    if case["paged"]:
        page, place = s["slots"] // PAGE, s["slots"] % PAGE
        s["kv"][page, s["layer"], 0, place] = k
        s["kv"][page, s["layer"], 1, place] = v
        return {"q": q, "kv": s["kv"]}
    return {"q": q, "kn": k, "vn": v.contiguous()}


def _decode(s):
    case, q = s["case"], s["q"]
    rows, heads, dim = q.shape
    kv_heads = case["kv_heads"]
    if own:
        from jeff_b200 import kernels

        return kernels.decode_attention(q, s["kv"], s["tables"], s["layer"], s["lengths"], FIXED, pr=s.get("pr"))
    pages = s["kv"][s["tables"][:, FIXED:].long(), s["layer"]].float()          # (rows, pages, 2, 32, heads, dim)
    keys, values = (pages[:, :, i].reshape(rows, -1, kv_heads, dim) for i in (0, 1))
    live = torch.arange(keys.shape[1], device="cuda") < s["lengths"][:, None]
    values = torch.where(live[:, :, None, None], values, 0.0)
    grouped = q.float().view(rows, kv_heads, heads // kv_heads, dim)
    scores = torch.einsum("rhgd,rjhd->rhgj", grouped, keys) / math.sqrt(dim)
    scores = torch.where(live[:, None, None], scores, -math.inf)
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    weights = weights / weights.sum(-1, keepdim=True)
    out = torch.einsum("rhgj,rjhd->rhgd", weights, values).reshape(rows, heads, dim)
    if not case["gated"]:
        return out.bfloat16()
    gate = s["pr"][:, :heads * 2 * dim].view(rows, heads, 2 * dim)[:, :, dim:].float()
    return (out / (1 + torch.exp(-gate))).bfloat16().view(rows, heads * dim)


def _scan(s):
    if own:
        from jeff_b200 import kernels

        o = kernels.linear_scan(s["q"], s["k"], s["v"], s["g"], s["pages"], s["tables"], s["layer"], real=s["real"],
                                out_tables=s["out_tables"])
        return {"o": o, "pages": s["pages"]}
    size = 64
    rows, tokens = s["q"].shape[:2]
    chunks = -(-tokens // size)
    live = torch.arange(chunks * size, device="cuda") < s["real"][:, None]

    def cut(x):   # (rows, tokens, heads, ...) -> (rows, heads, chunks, 64, ...), zeros past each row's end
        x = torch.nn.functional.pad(x, (0, 0) * (x.dim() - 2) + (0, chunks * size - tokens))
        x = torch.where(live.view(rows, -1, *[1] * (x.dim() - 2)), x, 0)
        return x.view(rows, chunks, size, *x.shape[2:]).movedim(3, 1)

    q, k, v = (cut(s[x].float()) for x in "qkv")
    # sums of decays in 64 bits: the factors are exponentials of their differences
    log = cut(s["g"].double().expand(rows, tokens, LIN_HEADS)).cumsum(-1)
    inner = torch.exp((log[..., :, None] - log[..., None, :]).tril()).tril().float()
    total = log[..., -1]                                                      # (rows, heads, chunks)
    grown = (k * torch.exp(total[..., None] - log).float()[..., None]).transpose(-1, -2) @ v
    upto = torch.nn.functional.pad(total.cumsum(-1), (1, 0))                   # decay ahead of each chunk, and in all
    carry = torch.exp((upto[..., :, None] - upto[..., None, 1:]).tril(-1)).tril(-1).float()   # (chunks + 1, chunks)
    page, slot = _state_at(s["tables"], s["layer"])
    begin = s["pages"][page, slot]
    states = torch.einsum("rhcd,rhdij->rhcij", carry, grown) + torch.exp(upto).float()[..., None, None] * begin[:, :, None]
    o = ((q @ k.transpose(-1, -2)) * inner) @ v + torch.exp(log).float()[..., None] * (q @ states[:, :, :-1])
    o = (o / math.sqrt(LIN_DIM)).movedim(1, 3).reshape(rows, chunks * size, LIN_HEADS, LIN_DIM)[:, :tokens]
    page, slot = _state_at(s["out_tables"], s["layer"])
    s["pages"][page, slot] = states[:, :, -1]
    return {"o": o.bfloat16(), "pages": s["pages"]}


def _step(s):
    if own:
        from jeff_b200 import kernels

        o = kernels.linear_step(s["q"], s["k"], s["v"], s["g"], s["pages"], s["tables"], s["layer"],
                                beta=s.get("beta"))
        return {"o": o, "pages": s["pages"]}
    page, slot = _state_at(s["tables"], s["layer"])
    q, k, v = (s[x].float() for x in "qkv")
    new = torch.exp(s["g"].expand(q.shape[:2]))[..., None, None] * s["pages"][page, slot]
    if "beta" in s:
        v = s["beta"].float()[..., None] * (v - (new * k[..., None]).sum(-2))
    new = new + k[..., None] * v[..., None, :]
    s["pages"][page, slot] = new
    return {"o": ((new * q[..., None]).sum(-2) / math.sqrt(LIN_DIM)).bfloat16(), "pages": s["pages"]}


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
    if case["op"] == "tables":
        rows = case["rows"]
        # which length meets which number of new tokens is the seed's: the pages taken are counted at the mean
        taken = rows * (case["new_lo"] + case["new_hi"]) / 2 / PAGE
        if case["fixed"]:
            taken += FIXED * (rows if case["hi"] == 0 else 1)
        return {"bytes": 8 * rows + 8 * taken + 16 * case["tokens"] + 8 * (rows + 1), "flops": 0}
    if case["op"] == "prep":
        t, values = case["tokens"], (HEADS + 2 * KV_HEADS) * DIM
        return {"bytes": t * (2 * 2 * values + 4 * case["axes"] + (8 if case["paged"] else 0)) + 8 * DIM,
                "flops": t * (HEADS + KV_HEADS) * (4 * DIM + 3 * ROT)}
    if case["op"] == "decode":
        cached = sum(_spread(case["rows"], case["lo"], case["hi"]))
        heads = case["rows"] * case["heads"] * case["dim"]
        return {"bytes": cached * case["kv_heads"] * case["dim"] * 2 * 2 + heads * 2 * (3 if case["gated"] else 2),
                "flops": cached * case["heads"] * case["dim"] * 4}
    states = case["rows"] * LIN_HEADS * LIN_DIM * LIN_DIM
    if case["op"] == "scan":
        real = sum(_spread(case["rows"], case["lo"], case["tokens"])) * LIN_HEADS
        padded = case["rows"] * case["tokens"] * LIN_HEADS
        # each token's part of the state and its read of it; its outputs past the row's end are zeros
        return {"bytes": 2 * LIN_DIM * (3 * real + padded) + (4 * real if case["per_token"] else 0) + 8 * states,
                "flops": real * 4 * LIN_DIM * LIN_DIM}
    heads = case["rows"] * LIN_HEADS
    return {"bytes": 8 * states + heads * (4 * 2 * LIN_DIM + 6), "flops": states * (8 if case["delta"] else 5)}


# ---------------------------------------------------------------- the definitions, in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "tables":
        return None
    if case["op"] == "prep":
        t = case["tokens"]
        wide = s["pr"].double()
        freq = s["inv_freq"].double()
        turns = torch.stack([s["positions"][a].double() * freq[i]
                             for i, a in enumerate(_axis_of(case["axes"], case["interleaved"]))], 1)
        spin = torch.polar(torch.ones_like(turns), turns)[:, None]

        def head(x, w1):
            x = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / DIM + EPS) * w1.double()
            z = torch.complex(x[..., :32].contiguous(), x[..., 32:64].contiguous()) * spin
            return torch.cat([z.real, z.imag, x[..., 64:]], -1)

        q = head(torch.stack([wide[:, 512 * h:512 * h + 256] for h in range(HEADS)], 1), s["q_w1"])
        k = head(wide[:, 4096:4608].reshape(t, 2, 256), s["k_w1"])
        v = wide[:, 4608:].reshape(t, 2, 256)
        if not case["paged"]:
            return {"q": q, "kn": k, "vn": v}
        kv = s["kv"].double()
        flat = kv.permute(0, 3, 1, 2, 4, 5).reshape(-1, LAYERS, 2, KV_HEADS, DIM)
        flat[s["slots"], s["layer"]] = torch.stack([k, v], 1)
        return {"q": q, "kv": flat.view(-1, PAGE, LAYERS, 2, KV_HEADS, DIM).permute(0, 2, 3, 1, 4, 5)}
    if case["op"] == "decode":
        group = case["heads"] // case["kv_heads"]
        out = torch.zeros(case["rows"], case["heads"], case["dim"], dtype=torch.float64, device="cuda")
        for r, n in enumerate(s["lengths"].tolist()):
            mine = s["tables"][r, FIXED:FIXED + _pages(n)].long()
            both = s["kv"][mine, s["layer"]].double().transpose(0, 1).reshape(2, -1, case["kv_heads"], case["dim"])
            for h in range(case["heads"]):
                p = torch.softmax(both[0, :n, h // group] @ s["q"][r, h].double() * case["dim"] ** -0.5, 0)
                out[r, h] = p @ both[1, :n, h // group]
        if not case["gated"]:
            return out
        gates = s["pr"][:, :2 * case["heads"] * case["dim"]].double().reshape(case["rows"], case["heads"], 2, -1)[:, :, 1]
        return (out * torch.sigmoid(gates)).flatten(1)
    page, slot = _state_at(s["tables"], s["layer"])
    memory = s["pages"][page, slot].double()
    pages = s["pages"].double()
    if case["op"] == "step":
        kept = torch.exp(s["g"].double()).expand(case["rows"], LIN_HEADS)[..., None, None] * memory
        k, v = s["k"].double(), s["v"].double()
        if case["delta"]:
            v = s["beta"].double()[..., None] * (v - torch.einsum("rhij,rhi->rhj", kept, k))
        memory = kept + torch.einsum("rhi,rhj->rhij", k, v)
        pages[page, slot] = memory
        return {"o": torch.einsum("rhij,rhi->rhj", memory, s["q"].double()) * LIN_DIM ** -0.5, "pages": pages}
    o = torch.zeros(*s["q"].shape, dtype=torch.float64, device="cuda")
    g = torch.exp(s["g"].double()).expand(case["rows"], case["tokens"], LIN_HEADS)
    q, k, v = (s[x].double() for x in "qkv")
    for t in range(case["tokens"]):
        live = (t < s["real"])[:, None, None, None]
        memory = torch.where(live, g[:, t, :, None, None] * memory + k[:, t, :, :, None] * v[:, t, :, None, :], memory)
        o[:, t] = torch.where(live[..., 0], (q[:, t, :, None, :] @ memory)[:, :, 0] * LIN_DIM ** -0.5, 0.0)
    page, slot = _state_at(s["out_tables"], s["layer"])
    pages[page, slot] = memory
    return {"o": o, "pages": pages}
