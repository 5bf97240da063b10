"""The operators around a decoder layer's attention, as cases to measure.

Four operators, each in a plain form (elementary torch operations in 32 bits) and, with ``own`` set, as the calls that a
user makes of ``klearu_b200.attention`` and ``klearu_b200.quant``:

* ``append``  rotary positions on queries and keys, keys and values written to a paged cache of 4-bit codes;
* ``attend``  attention of new tokens over that cache;
* ``norm``    residual addition, root-mean-square norm and 8-bit codes with a scale for each row;
* ``matmul``  the product of two matrices of 8-bit codes with a scale for each row and each output channel.

A cached head vector x of D values is held as codes c in 0..15 with x ~ s * c + m, where m = bf16(min x),
s = bf16((max x - min x) / 15) and c = clamp(rint((x - m) / s), 0, 15), or 0 where s is 0.
"""

import math

import torch

own = False

DEV = "cuda:0"

# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------


def listed():
    return [
        # one token of a 32-head model with as many key heads: the call of every decode step, where latency counts
        {"name": "append one token", "op": "append", "seqs": 1, "q_min": 1, "q_max": 1, "ctx_max": 777, "heads": 32, "kv_heads": 32,
         "dim": 128, "page": 16, "rot": 128, "interleaved": False, "factor": 1.0},
        # ragged prompts at far positions with frequencies stretched for a long context, half of each head rotated
        {"name": "append prompts", "op": "append", "seqs": 5, "q_min": 1500, "q_max": 4500, "ctx_max": 65536, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 64, "rot": 64, "interleaved": True, "factor": 8.0},
        # one token over a short context: latency of the smallest decode step
        {"name": "attend one token", "op": "attend", "seqs": 1, "q_min": 1, "q_max": 1, "ctx_max": 777, "heads": 32, "kv_heads": 32,
         "dim": 128, "page": 16, "window": 0},
        # a serving batch, one token each, contexts of all lengths: bound by reading the cache
        {"name": "attend batch of 64", "op": "attend", "seqs": 64, "q_min": 1, "q_max": 1, "ctx_max": 16384, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 64, "window": 0},
        # one token over a very long context: few rows, a long axis to split
        {"name": "attend long context", "op": "attend", "seqs": 1, "q_min": 1, "q_max": 1, "ctx_max": 131071, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 32, "window": 0},
        # a few drafted tokens for each sequence, small heads, a sliding window, an odd group
        {"name": "attend drafts", "op": "attend", "seqs": 9, "q_min": 1, "q_max": 7, "ctx_max": 5000, "heads": 15, "kv_heads": 5,
         "dim": 64, "page": 48, "window": 1024},
        # ragged prompt chunks after earlier context: bound by the matrix products
        {"name": "attend prompts", "op": "attend", "seqs": 4, "q_min": 1000, "q_max": 3000, "ctx_max": 6000, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 64, "window": 0},
        # the hidden state of one token, 32 bits, before a layer's projections
        {"name": "norm one row", "op": "norm", "rows": 1, "cols": 4096, "type": "f32"},
        # a prompt's rows: 16-bit block outputs added to the 32-bit residual
        {"name": "norm prompt", "op": "norm", "rows": 8191, "cols": 4096, "type": "bf16"},
        # one token through the three projections before attention
        {"name": "matmul one row", "op": "matmul", "rows": 1, "k": 4096, "n": 12288, "type": "bf16"},
        # a decode batch through a down projection
        {"name": "matmul batch of 33", "op": "matmul", "rows": 33, "k": 11008, "n": 4096, "type": "f32"},
        # a prompt through an up projection
        {"name": "matmul prompt", "op": "matmul", "rows": 8191, "k": 4096, "n": 11008, "type": "bf16"},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "norm", "matmul"])
    if op == "norm":
        rows = _log_int(rng, 1, 8191)
        return {"op": op, "rows": rows, "cols": _log_int(rng, 64, 11008), "type": rng.choice(["f32", "bf16"])}
    if op == "matmul":
        return {"op": op, "rows": _log_int(rng, 1, 6000), "k": _log_int(rng, 64, 11008), "n": _log_int(rng, 16, 4096),
                "type": rng.choice(["f32", "bf16"])}
    kv_heads = rng.randint(1, 8)
    group = rng.choice([1, 2, 3, 4, 6, 7, 8])
    dim = rng.choice([64, 128])
    page = 16 * rng.randint(1, 8)
    if op == "append":
        rot = rng.choice([None, dim, dim // 2, dim // 4 + 2])
        q_max = _log_int(rng, 1, 2000)
        return {"op": op, "seqs": _log_int(rng, 1, 12), "q_min": rng.randint(1, q_max), "q_max": q_max, "ctx_max": _log_int(rng, q_max, 60000),
                "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "page": page, "rot": rot or 0, "interleaved": rng.random() < 0.5,
                "factor": rng.choice([1.0, 4.0])}
    window = rng.choice([0, 0, rng.randint(1, 3000)])
    if rng.random() < 0.5:  # decode steps and drafts
        q_max = rng.choice([1, 1, rng.randint(2, 12)])
        seqs = _log_int(rng, 1, 100)
        ctx = _log_int(rng, q_max, max(q_max, min(131071, 400000 // seqs)))
    else:  # prompt chunks
        q_max = _log_int(rng, 13, 2000)
        seqs = rng.randint(1, 4)
        ctx = _log_int(rng, q_max, 6000)
    return {"op": op, "seqs": seqs, "q_min": rng.randint(1, q_max), "q_max": q_max, "ctx_max": ctx, "heads": kv_heads * group,
            "kv_heads": kv_heads, "dim": dim, "page": page, "window": window}


def _lens(case):
    """New tokens and context (new ones included) of each sequence: spread over the case's range by a fixed low-discrepancy sequence."""
    n = case["seqs"]
    q, kv = [], []
    for i in range(n):
        a, b = (0.5 + i * 0.6180339887498949) % 1.0, (1.0 - i * 0.7548776662466927) % 1.0 or 1.0
        ql = case["q_min"] + int(a * (case["q_max"] - case["q_min"] + 1))
        ql = min(ql, case["q_max"])
        q.append(ql)
        kv.append(max(ql, int(round(b * case["ctx_max"]))) if n > 1 else max(ql, case["ctx_max"]))
    return q, kv


def work(case):
    if case["op"] == "norm":
        n = case["rows"] * case["cols"]
        return {"bytes": n * ((4 if case["type"] == "f32" else 2) + 4 + 4 + 1) + 4 * (case["cols"] + case["rows"]), "flops": 8 * n}
    if case["op"] == "matmul":
        m, k, n = case["rows"], case["k"], case["n"]
        return {"bytes": m * k + n * k + 4 * (m + n) + m * n * (4 if case["type"] == "f32" else 2), "flops": 2 * m * n * k}
    q, kv = _lens(case)
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    held = hk * (d + 8)  # bytes of a token's codes, steps and minima of keys and values
    if case["op"] == "append":
        t = sum(q)
        table = 4 * case["rot"] * t
        # q, k, v read; q and the cache written; the cached values read back
        return {"bytes": t * (4 * hq * d + 4 * hk * d + 2 * held + 4 * hk * d) + table, "flops": t * (3 * hq * d + 20 * hk * d)}
    w = case["window"]
    seen = pairs = 0
    for a, b in zip(q, kv):
        first = b - a
        seen += b if not w else min(b, a + w - 1)
        pairs += sum(min(p + 1, w) for p in range(first, b)) if w else a * (first + 1 + b) // 2
    return {"bytes": seen * held + sum(q) * hq * d * 4, "flops": 4 * pairs * hq * d}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _pages(case, g):
    """Context lengths and each sequence's pages, in an order of chance."""
    q, kv = _lens(case)
    page = case["page"]
    need = [-(-n // page) for n in kv]
    wide = max(need)
    order = torch.randperm(sum(need), generator=g, device=DEV).to(torch.int32)
    table = torch.zeros(len(kv), wide, dtype=torch.int32, device=DEV)
    row = torch.repeat_interleave(torch.arange(len(kv), device=DEV), torch.tensor(need, device=DEV))
    col = torch.cat([torch.arange(n, device=DEV) for n in need])
    table[row, col] = order
    return q, kv, table, sum(need)


def _cu(lens):
    return torch.tensor([0] + lens, dtype=torch.int64).cumsum(0).to(torch.int32).to(DEV)


def _keys(g, t, heads, dim):
    """Keys with channels of their own offset and size, as projections give them, and plain values."""
    k = torch.randn(t, heads, dim, generator=g, device=DEV, dtype=torch.bfloat16)
    size = torch.exp(0.5 * torch.randn(heads, dim, generator=g, device=DEV)).bfloat16()
    k = k.mul_(size).add_(torch.randn(heads, dim, generator=g, device=DEV).bfloat16())
    return k, torch.randn(t, heads, dim, generator=g, device=DEV, dtype=torch.bfloat16)


def _inputs(case, seed):
    g = _gen(seed)
    if case["op"] == "norm":
        m, n = case["rows"], case["cols"]
        x = torch.randn(m, n, generator=g, device=DEV)
        x = x if case["type"] == "f32" else x.bfloat16()
        residual = 4 * torch.randn(m, n, generator=g, device=DEV)
        return {"x": x, "residual": residual, "weight": 1 + 0.2 * torch.randn(n, generator=g, device=DEV)}
    if case["op"] == "matmul":
        m, k, n = case["rows"], case["k"], case["n"]
        pad = -(-k // 16) * 16  # rows of codes start on 16 bytes, as the norm writes them
        a = torch.randint(-127, 128, (m, pad), generator=g, device=DEV, dtype=torch.int8)[:, :k]
        w = torch.randint(-127, 128, (n, k), generator=g, device=DEV, dtype=torch.int8)
        return {"a": a, "w": w, "a_scale": 0.01 + 0.05 * torch.rand(m, generator=g, device=DEV),
                "w_scale": 0.0002 + 0.001 * torch.rand(n, generator=g, device=DEV)}
    q_len, kv_len, table, pages = _pages(case, g)
    t = sum(q_len)
    d = {"q_len": q_len, "kv_len": kv_len, "table": table, "pages": pages, "cu": _cu(q_len),
         "kv": torch.tensor(kv_len, dtype=torch.int32, device=DEV)}
    if case["op"] == "append":
        hq, hk, dim = case["heads"], case["kv_heads"], case["dim"]
        # one projection's output holds queries, keys and values side by side
        qkv = torch.randn(t, (hq + 2 * hk) * dim, generator=g, device=DEV, dtype=torch.bfloat16)
        d["q"], d["k"], d["v"] = (x.unflatten(1, (-1, dim)) for x in qkv.split([hq * dim, hk * dim, hk * dim], 1))
        return d
    d["q"] = torch.randn(t, case["heads"], case["dim"], generator=g, device=DEV, dtype=torch.bfloat16)
    d["k"], d["v"] = _keys(g, sum(kv_len), case["kv_heads"], case["dim"])
    return d


def _frequencies(case):
    """Angles per position, in 64 bits: base^(-2i/rot), those of few turns over 8192 positions divided by the factor."""
    rot = case["rot"]
    inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if case["factor"] != 1.0:
        turns = 8192 * inv / (2 * math.pi)
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        inv = inv * (keep + (1 - keep) / case["factor"])
    return inv


def _attention_factor(case):
    return 0.1 * math.log(case["factor"]) + 1.0


# ---------------------------------------------------------------------------
# What a program has in hand before the call
# ---------------------------------------------------------------------------


def _token_rows(lens):
    """For each token of ragged sequences: its sequence and its place in it."""
    n = torch.tensor(lens, device=DEV)
    seq = torch.repeat_interleave(torch.arange(len(lens), device=DEV), n)
    start = torch.cumsum(n, 0) - n
    return seq, torch.arange(int(n.sum()), device=DEV) - start[seq]


def _slots(d, page, seq, index):
    return d["table"][seq, index // page].long() * page + index % page


def prepare(case, seed):
    d = _inputs(case, seed)
    s = {"case": case, **d}
    if case["op"] == "norm":
        return s
    if case["op"] == "matmul":
        if own:
            from klearu_b200.quant import Q8Linear

            s["linear"] = Q8Linear(d["w"], d["w_scale"])
        return s
    hk, dim, page = case["kv_heads"], case["dim"], case["page"]
    if own:
        from klearu_b200.attention import Kv4Cache, RopeTable, SeqBatch

        s["cache"] = Kv4Cache(d["pages"], page, hk, dim)
        s["batch"] = SeqBatch(d["cu"], d["kv"], d["table"], max_q=max(d["q_len"]), max_kv=max(d["kv_len"]))
        if case["op"] == "attend":
            every = SeqBatch(_cu(d["kv_len"]), d["kv"], d["table"], max_q=max(d["kv_len"]), max_kv=max(d["kv_len"]))
            s["cache"].append(s.pop("k"), s.pop("v"), every)
        elif case["rot"]:
            scaling = {} if case["factor"] == 1.0 else {"scaling": "by_parts", "factor": case["factor"], "original_positions": 8192,
                                                        "low_turns": 1.0, "high_turns": 4.0}
            s["rope"] = RopeTable(case["rot"], max(d["kv_len"]), base=10000.0, interleaved=case["interleaved"],
                                  attention_factor=_attention_factor(case), **scaling)
        return s
    seq, index = _token_rows(d["q_len"])
    s["seq"] = seq
    s["first"] = d["kv"].long() - torch.tensor(d["q_len"], device=DEV)  # new tokens follow this much context
    s["position"] = s["first"][seq] + index
    slots = d["pages"] * page
    for x in ("k", "v"):
        s["cache_" + x] = torch.zeros(slots, hk, dim, dtype=torch.uint8, device=DEV)
        s["step_" + x], s["low_" + x] = (torch.zeros(slots, hk, 1, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    if case["op"] == "append":
        s["slots"] = _slots(d, page, seq, s["position"])
        if case["rot"]:
            angle = torch.arange(max(d["kv_len"]), dtype=torch.float64, device=DEV)[:, None] * _frequencies(case).to(DEV)
            f = _attention_factor(case)
            s["cos"], s["sin"] = (angle.cos() * f).float(), (angle.sin() * f).float()
        return s
    kv_seq, kv_index = _token_rows(d["kv_len"])
    at = _slots(d, page, kv_seq, kv_index)
    for x in ("k", "v"):
        rows = s.pop(x)
        for i in range(0, len(rows), 1 << 16):
            part = slice(i, i + (1 << 16))
            s["cache_" + x][at[part]], s["step_" + x][at[part]], s["low_" + x][at[part]] = _plain_codes(rows[part].float())
    b, wide = len(d["kv_len"]), max(d["kv_len"])
    place = torch.arange(wide, device=DEV).expand(b, wide)
    s["kv_slots"] = _slots(d, page, torch.arange(b, device=DEV)[:, None], place)  # behind a sequence's end: a page of chance, masked
    s["row"] = index
    return s


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------


def _plain_codes(x):
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    step, low = ((high - low) / 15).bfloat16(), low.bfloat16()
    code = torch.where(step > 0, ((x - low.float()) / step.float()).round(), 0.0).clamp(0, 15)
    return code.to(torch.uint8), step, low


def _plain_rotate(x, cos, sin, rot, interleaved):
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
    else:
        a, b = x[..., : rot // 2], x[..., rot // 2 : rot]
    u, v = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([u, v], -1).flatten(-2) if interleaved else torch.cat([u, v], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _plain_append(s):
    c = s["case"]
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    if c["rot"]:
        cos, sin = s["cos"][s["position"]][:, None], s["sin"][s["position"]][:, None]
        q = _plain_rotate(q, cos, sin, c["rot"], c["interleaved"])
        k = _plain_rotate(k, cos, sin, c["rot"], c["interleaved"])
    out = {"q": q.bfloat16()}
    for name, x in (("k", k), ("v", v)):  # the two tensors of the cache
        s["cache_" + name][s["slots"]], s["step_" + name][s["slots"]], s["low_" + name][s["slots"]] = _plain_codes(x)
        out[name] = _plain_values(s, name, s["slots"]).bfloat16()
    return out


def _plain_values(s, name, at):
    return s["cache_" + name][at].float() * s["step_" + name][at].float() + s["low_" + name][at].float()


def _plain_attend(s):
    c = s["case"]
    hq, hk, dim = c["heads"], c["kv_heads"], c["dim"]
    group = hq // hk
    b, wide = s["kv_slots"].shape
    rows = max(s["q_len"])
    q = torch.zeros(b, rows, hq, dim, device=DEV)
    q[s["seq"], s["row"]] = s["q"].float()
    q = q.view(b, rows, hk, group, dim).permute(0, 2, 3, 1, 4).reshape(b * hk, group * rows, dim)
    k = _plain_values(s, "k", s["kv_slots"]).transpose(1, 2).reshape(b * hk, wide, dim)
    score = torch.bmm(q, k.transpose(1, 2)).view(b, hk, group, rows, wide) * dim**-0.5
    del k
    at = s["first"][:, None] + torch.arange(rows, device=DEV)
    place = torch.arange(wide, device=DEV)
    seen = (place[None, None] <= at[:, :, None]) & (place[None, None] < s["kv"][:, None, None])
    if c["window"]:
        seen &= place[None, None] > at[:, :, None] - c["window"]
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(top.isfinite(), top, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    v = _plain_values(s, "v", s["kv_slots"]).transpose(1, 2).reshape(b * hk, wide, dim)
    o = torch.bmm(p.view(b * hk, group * rows, wide), v).view(b, hk, group, rows, dim)
    o = torch.where(total > 0, o / total, 0.0)
    return o.permute(0, 3, 1, 2, 4).reshape(b, rows, hq, dim)[s["seq"], s["row"]].bfloat16()


def _plain_norm(s):
    h = s["x"].float() + s["residual"]
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-5)
    # the row's factor cancels in the codes: 64 bits, so that values next to a border fall on the right side of it
    u = h.double() * s["weight"].double()
    top = u.abs().amax(-1, keepdim=True)
    code = torch.where(top > 0, (u * 127 / top).round(), 0.0)
    scale = (y * s["weight"]).abs().amax(-1) / 127
    return {"hidden": h, "scale": scale, "values": code.float() * scale[:, None]}


def _plain_matmul(s):
    # 64 bits: sums of products of 8-bit codes pass 24 bits
    total = (s["a"].double() @ s["w"].double().T).float()
    out = total * s["a_scale"][:, None] * s["w_scale"]
    return out if s["case"]["type"] == "f32" else out.bfloat16()


def run(s):
    op = s["case"]["op"]
    if not own:
        return {"append": _plain_append, "attend": _plain_attend, "norm": _plain_norm, "matmul": _plain_matmul}[op](s)
    if op == "append":
        q = s["cache"].append(s["k"], s["v"], s["batch"], q=s["q"], rope=s.get("rope"))
        k, v = s["cache"].read(s["batch"], len(s["k"]))
        return {"q": q, "k": k, "v": v}
    if op == "attend":
        return s["cache"].attend(s["q"], s["batch"], window=s["case"]["window"])
    if op == "norm":
        from klearu_b200.quant import add_rms_norm_q8

        r = add_rms_norm_q8(s["x"], s["weight"], residual=s["residual"], eps=1e-5)
        return {"hidden": r.hidden, "scale": r.scales, "values": r.codes * r.scales[:, None]}
    return s["linear"].forward(s["a"], s["a_scale"], out_dtype=torch.float32 if s["case"]["type"] == "f32" else torch.bfloat16)


# ---------------------------------------------------------------------------
# The definitions, in 64 bits
# ---------------------------------------------------------------------------


def _exact_held(x):
    """The values that a head vector's 4-bit codes stand for."""
    x = x.double()
    lo, hi = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
    s, m = ((hi - lo) / 15).to(torch.bfloat16).double(), lo.to(torch.bfloat16).double()
    c = torch.nan_to_num((x - m) / s, nan=0.0, posinf=0.0, neginf=0.0).round().clamp(0, 15)
    return c * s + m


def _exact_append(case, d):
    rot = case["rot"]
    at = torch.cat([torch.arange(b - a, b, dtype=torch.float64) for a, b in zip(d["q_len"], d["kv_len"])]).to(DEV)

    def turn(x):
        x = x.double()
        if not rot:
            return x
        z = torch.outer(at, _frequencies(case).to(DEV))
        f = _attention_factor(case)
        cos, sin = (z.cos() * f).float().double()[:, None], (z.sin() * f).float().double()[:, None]  # the table holds 32 bits
        first = torch.arange(0, rot, 2, device=DEV) if case["interleaved"] else torch.arange(rot // 2, device=DEV)
        second = first + (1 if case["interleaved"] else rot // 2)
        y = x.clone()
        y[..., first] = x[..., first] * cos - x[..., second] * sin
        y[..., second] = x[..., second] * cos + x[..., first] * sin
        return y

    return {"q": turn(d["q"]), "k": _exact_held(turn(d["k"])), "v": _exact_held(d["v"])}


def _exact_attend(case, d):
    if work(case)["flops"] > 2e12:
        return None
    group = case["heads"] // case["kv_heads"]
    out, a, b = [], 0, 0
    for ql, kl in zip(d["q_len"], d["kv_len"]):
        q = d["q"][a : a + ql].double()
        k, v = _exact_held(d["k"][b : b + kl]), _exact_held(d["v"][b : b + kl])
        i = torch.arange(kl - ql, kl, device=DEV)[:, None]
        j = torch.arange(kl, device=DEV)
        hide = j > i
        if case["window"]:
            hide = hide | (j <= i - case["window"])
        o = torch.empty(ql, case["heads"], case["dim"], dtype=torch.float64, device=DEV)
        for h in range(case["heads"]):
            z = (q[:, h] @ k[:, h // group].T / math.sqrt(case["dim"])).masked_fill(hide, -math.inf)
            o[:, h] = torch.softmax(z, -1) @ v[:, h // group]
        out.append(o)
        a, b = a + ql, b + kl
    return torch.cat(out)


def _exact_norm(d):
    h = (d["x"].float() + d["residual"]).double()  # the residual stream is held in 32 bits
    y = h / (h.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt() * d["weight"].double()
    top = y.abs().max(-1, keepdim=True).values
    u = h * d["weight"].double()
    code = (u / u.abs().max(-1, keepdim=True).values * 127).round()
    return {"hidden": h, "scale": top[:, 0] / 127, "values": code * top / 127}


def exact(case, seed):
    d = _inputs(case, seed)
    if case["op"] == "append":
        return _exact_append(case, d)
    if case["op"] == "attend":
        return _exact_attend(case, d)
    if case["op"] == "norm":
        return _exact_norm(d)
    total = torch.mm(d["a"].double(), d["w"].double().t())
    return total * torch.outer(d["a_scale"].double(), d["w_scale"].double())
