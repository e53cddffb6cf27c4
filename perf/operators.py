"""The serving operators of the LM, as they are timed: rotary positions, the append to a paged 4-bit KV cache, attention over
that cache and the rules applied to logits before a token is sampled. Each has a plain form in torch and the call of this
framework."""
import math
import os
import sys

import numpy as np
import torch

own = False
_ACB = None
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _acb():
    global _ACB
    if _ACB is None:
        p = os.path.join(os.getcwd(), "hbd-acestep.cpp_b200")
        if p not in sys.path:
            sys.path.insert(0, p)
        import acb
        _ACB = acb
    return _ACB


def listed():
    return [
        # q and k of one decode step of 8 sequences at the LM's shape (16 + 8 heads of 128)
        {"name": "rope decode", "op": "rope", "n_tok": 8, "heads": 24, "dim": 128, "rope_dim": 128, "layout": "half",
         "dtype": "f32", "max_pos": 8192, "inverse": False},
        # a batch of prompts with far positions, a part of a wider head rotated, interleaved pairs
        {"name": "rope prompt", "op": "rope", "n_tok": 8191, "heads": 24, "dim": 192, "rope_dim": 64, "layout": "interleaved",
         "dtype": "bf16", "max_pos": 131072, "inverse": False},
        # one decode step of 8 sequences: q rotated, k and v into their pages
        {"name": "append decode", "op": "append", "n_seq": 8, "q_lo": 1, "q_hi": 1, "past": 1500, "heads": 16, "kv_heads": 8,
         "dim": 128, "rope_dim": 128, "layout": "half", "dtype": "f32", "page": 64, "norm": True},
        # prompts of many lengths at the LM's shape
        {"name": "append prompts", "op": "append", "n_seq": 16, "q_lo": 37, "q_hi": 2048, "past": 0, "heads": 16,
         "kv_heads": 8, "dim": 128, "rope_dim": 128, "layout": "half", "dtype": "bf16", "page": 64, "norm": True},
        # chunks behind a past, no norms, short heads rotated in part, small pages
        {"name": "append chunks", "op": "append", "n_seq": 5, "q_lo": 100, "q_hi": 777, "past": 333, "heads": 14,
         "kv_heads": 2, "dim": 64, "rope_dim": 32, "layout": "interleaved", "dtype": "f16", "page": 16, "norm": False},
        # one sequence behind a prompt of 512 and 1024 new tokens: latency
        {"name": "attn one", "op": "attn", "n_seq": 1, "q_lo": 1, "q_hi": 1, "kv_lo": 1536, "kv_hi": 1536, "heads": 16,
         "kv_heads": 8, "dim": 128, "dtype": "f32", "page": 64, "window": 0},
        # a served batch with lengths of every size up to the LM's 8192
        {"name": "attn batch", "op": "attn", "n_seq": 96, "q_lo": 1, "q_hi": 1, "kv_lo": 200, "kv_hi": 8192, "heads": 32,
         "kv_heads": 8, "dim": 128, "dtype": "bf16", "page": 64, "window": 0},
        # two very long sequences: the keys are split
        {"name": "attn long", "op": "attn", "n_seq": 2, "q_lo": 1, "q_hi": 1, "kv_lo": 131071, "kv_hi": 131071, "heads": 16,
         "kv_heads": 8, "dim": 128, "dtype": "f16", "page": 128, "window": 0},
        # a few drafted tokens each, short heads, a window, small pages, seven query heads to a kv head
        {"name": "attn drafts", "op": "attn", "n_seq": 24, "q_lo": 1, "q_hi": 7, "kv_lo": 50, "kv_hi": 4000, "heads": 14,
         "kv_heads": 2, "dim": 64, "dtype": "f16", "page": 16, "window": 1000},
        # chunks of prompts over what is cached of them
        {"name": "attn prompts", "op": "attn", "n_seq": 4, "q_lo": 1200, "q_hi": 2048, "kv_lo": 2048, "kv_hi": 5000,
         "heads": 16, "kv_heads": 8, "dim": 128, "dtype": "bf16", "page": 64, "window": 0},
        # one sequence, everything on: latency
        {"name": "logits one", "op": "logits", "rows": 1, "vocab": 217472, "dtype": "f32", "out": "f32", "hist": 1536,
         "bias": 20, "masks": 1},
        # a served batch of 16-bit logits, long histories, a grammar for every second row
        {"name": "logits batch", "op": "logits", "rows": 128, "vocab": 151936, "dtype": "bf16", "out": "f32", "hist": 4100,
         "bias": 300, "masks": 7},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the same ranges that costs no more than the largest listed one"""
    most = [max(work(c)[k] for c in listed()) for k in ("bytes", "flops")]
    while True:
        case = _any(rng)
        w = work(case)
        if w["bytes"] <= most[0] and w["flops"] <= most[1]:
            return case


def _any(rng):
    op = rng.choice(["rope", "append", "attn", "attn", "logits"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "rope":
        dim = 2 * rng.randint(16, 128)
        return {"op": op, "n_tok": _log(rng, 1, 8000), "heads": rng.randint(1, 40), "dim": dim,
                "rope_dim": rng.choice([dim, 2 * rng.randint(1, dim // 2)]), "layout": rng.choice(["half", "interleaved"]),
                "dtype": dtype, "max_pos": _log(rng, 8000, 131072), "inverse": rng.random() < 0.3}
    if op == "logits":
        return {"op": op, "rows": _log(rng, 1, 96), "vocab": _log(rng, 1000, 217472), "dtype": dtype,
                "out": rng.choice(["f32", dtype]), "hist": _log(rng, 1, 8000), "bias": rng.choice([0, _log(rng, 1, 300)]),
                "masks": rng.randint(0, 5)}
    dim, kv_heads = rng.choice([64, 128, 128, 256]), rng.choice([1, 2, 3, 4, 8])
    case = {"op": op, "heads": kv_heads * rng.randint(1, 9), "kv_heads": kv_heads, "dim": dim, "dtype": dtype,
            "page": rng.choice([16, 32, 64, 128, 256])}
    if op == "append":
        q_hi = _log(rng, 1, 1500)
        case.update(n_seq=rng.randint(1, 12), q_lo=rng.randint(1, q_hi), q_hi=q_hi, past=_log(rng, 1, 8000),
                    rope_dim=rng.choice([dim, dim // 2, 2 * rng.randint(1, dim // 2)]),
                    layout=rng.choice(["half", "interleaved"]), norm=rng.random() < 0.5)
        return case
    kind = rng.choice(["decode", "decode", "drafts", "prompts"])
    q_hi = {"decode": 1, "drafts": rng.randint(2, 12), "prompts": _log(rng, 30, 1000)}[kind]
    n_seq = _log(rng, 1, 64) if kind != "prompts" else rng.randint(1, 4)
    kv_hi = max(q_hi, _log(rng, 1, 40000 if n_seq <= 8 and q_hi < 30 else 4000))
    case.update(n_seq=n_seq, q_lo=rng.randint(1, q_hi), q_hi=q_hi, kv_lo=rng.randint(q_hi, kv_hi), kv_hi=kv_hi,
                window=rng.choice([0, 0, _log(rng, 1, 2000)]))
    return case


# ---- inputs -----------------------------------------------------------------------------------------

def _spread(n, lo, hi, step):
    """n lengths over [lo, hi], the last one hi: the case alone fixes them"""
    return [lo + int((hi - lo) * ((i + 1) * step % 1.0)) for i in range(n - 1)] + [hi]


def _lens(case):
    q = _spread(case["n_seq"], case["q_lo"], case["q_hi"], 0.61803)
    if case["op"] == "append":
        return q, [x + case["past"] for x in q]
    return q, _spread(case["n_seq"], case["kv_lo"], case["kv_hi"], 0.75488)


def _table(max_pos, rope_dim, dev, factor=8.0):
    """Rows (cos, sin) of each pair: base 1e6, positions divided by `factor` as for a context longer than the trained one"""
    i = torch.arange(rope_dim // 2, dtype=torch.float64, device=dev)
    a = torch.arange(max_pos, dtype=torch.float64, device=dev)[:, None] / factor * 1e6 ** (-2.0 * i / rope_dim)
    return torch.stack([a.cos(), a.sin()], -1).reshape(max_pos, rope_dim).float()


def _pages(case, kv_len, gen, dev, fill):
    """A pool with some pages to spare, the sequences' pages anywhere in it; `fill`: codes and scales of keys and values"""
    P, Nkv, D = case["page"], case["kv_heads"], case["dim"]
    need = [-(-n // P) for n in kv_len]
    n_pages = sum(need) + 3
    ids = torch.randperm(n_pages, generator=gen, device=dev).int()
    table = torch.full((len(need), max(need)), -1, dtype=torch.int32, device=dev)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = ids[at:at + n]
        at += n
    c = {"table": table}
    for n in ("k", "v"):
        if fill:
            c[n + "c"] = torch.randint(0, 256, (n_pages, Nkv, P, D // 2), dtype=torch.uint8, generator=gen, device=dev)
            d = 0.05 + 0.15 * torch.rand((n_pages, Nkv, P, D // 32), generator=gen, device=dev)
            c[n + "s"] = (d * (1 if n == "v" else 1.5)).bfloat16().half()
        else:
            c[n + "c"] = torch.zeros((n_pages, Nkv, P, D // 2), dtype=torch.uint8, device=dev)
            c[n + "s"] = torch.zeros((n_pages, Nkv, P, D // 32), dtype=torch.float16, device=dev)
    return c


def prepare(case, seed):
    dev = "cuda" if torch.cuda.is_available() else "cpu"
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    st = {"case": case}
    op = case["op"]
    rnd = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    if op == "rope":
        st["x"] = rnd(case["n_tok"], case["heads"], case["dim"]).to(TYPES[case["dtype"]])
        st["pos"] = torch.randint(0, case["max_pos"], (case["n_tok"],), generator=g, device=dev).int()
        st["rope"] = _table(case["max_pos"], case["rope_dim"], dev)
        st["out"] = torch.empty_like(st["x"])
        return st
    if op == "logits":
        R, V, L = case["rows"], case["vocab"], case["hist"]
        st["x"] = (rnd(R, V) * 3).to(TYPES[case["dtype"]])
        # tokens come again: half of a history is drawn from a few hundred
        few = torch.randint(0, V, (300,), generator=g, device=dev)
        st["hist"] = torch.where(torch.rand((R, L), generator=g, device=dev) < 0.5,
                                 few[torch.randint(0, 300, (R, L), generator=g, device=dev)],
                                 torch.randint(0, V, (R, L), generator=g, device=dev)).int()
        st["hist_len"] = torch.tensor(_spread(R, (L + 1) // 2, L, 0.61803), dtype=torch.int32, device=dev)
        st["prompt_len"] = st["hist_len"] // 3
        st["rep"] = 1 + 0.3 * torch.rand(R, generator=g, device=dev)
        st["freq"] = 0.2 * torch.rand(R, generator=g, device=dev)
        st["pres"] = 0.5 * torch.rand(R, generator=g, device=dev)
        if case["bias"]:
            st["bias_ids"] = torch.randint(0, V, (R, case["bias"]), generator=g, device=dev).int()
            st["bias_val"] = rnd(R, case["bias"]) * 2
        if case["masks"]:
            # one grammar state leaves few tokens, another most: bits set with a share of its own
            share = torch.rand((case["masks"], 1), generator=g, device=dev)
            bits = torch.rand((case["masks"], -(-V // 32) * 32), generator=g, device=dev) < share
            w = bits.view(case["masks"], -1, 32).long() << torch.arange(32, device=dev)
            w = w.sum(-1)
            st["mask"] = torch.where(w >= 2 ** 31, w - 2 ** 32, w).int()
            r = torch.arange(R, device=dev)
            st["mask_row"] = torch.where(r % 2 == 0, r // 2 % case["masks"], -1).int()
        st["out"] = torch.empty((R, V), dtype=TYPES[case["out"]], device=dev)
        return st
    q_len, kv_len = _lens(case)
    H, Nkv, D, T = case["heads"], case["kv_heads"], case["dim"], sum(q_len)
    st.update(_pages(case, kv_len, g, dev, op == "attn"))
    st["q_start"] = torch.tensor([0] + torch.tensor(q_len).cumsum(0).tolist(), dtype=torch.int32, device=dev)
    st["kv_len"] = torch.tensor(kv_len, dtype=torch.int32, device=dev)
    st["max_q"], st["max_kv"] = max(q_len), max(kv_len)
    if op == "append":
        st["qkv"] = rnd(T, (H + 2 * Nkv) * D).to(TYPES[case["dtype"]])
        st["seq"] = torch.cat([torch.full((n,), s) for s, n in enumerate(q_len)]).int().to(dev)
        st["pos"] = torch.cat([torch.arange(m - n, m) for n, m in zip(q_len, kv_len)]).int().to(dev)
        st["rope"] = _table(max(kv_len), case["rope_dim"], dev)
        st["q_norm"] = 1 + 0.1 * rnd(D) if case["norm"] else None
        st["k_norm"] = 1 + 0.1 * rnd(D) if case["norm"] else None
        st["out"] = torch.empty((T, H, D), dtype=TYPES[case["dtype"]], device=dev)
        st["k_out"] = torch.empty((T, Nkv, D), dtype=torch.float16, device=dev)
        st["v_out"] = torch.empty_like(st["k_out"])
    else:
        st["q"] = rnd(T, H, D).to(TYPES[case["dtype"]])
        st["out"] = torch.empty_like(st["q"])
    if own:  # what a server makes once: the handle on its cache and the workspace
        st["cache"] = _acb().KVCacheQ4(st["kc"], st["ks"], st["vc"], st["vs"], st["table"])
        if op == "attn":
            st["work"] = st["cache"].attn_workspace(T, H, st["max_q"], st["max_kv"])
    return st


# ---- plain forms -------------------------------------------------------------------------------------

def _rotate(x, pos, table, layout, inverse=False):
    """x [T, H, D]: the first table-width elements of every head rotated"""
    R = table.shape[1]
    c, s = table[pos.long(), 0::2][:, None], table[pos.long(), 1::2][:, None]
    if inverse:
        s = -s
    a, b = (x[..., 0:R // 2], x[..., R // 2:R]) if layout == "half" else (x[..., 0:R:2], x[..., 1:R:2])
    u, v = a * c - b * s, a * s + b * c
    y = torch.cat([u, v], -1) if layout == "half" else torch.stack([u, v], -1).flatten(-2)
    return torch.cat([y, x[..., R:]], -1)


def _norm(x, w, eps=1e-6):
    if w is None:
        return x
    mean = ((x * x).double().sum(-1, keepdim=True) / x.shape[-1]).float()
    return x * (1.0 / (mean + eps).sqrt()) * w


def _to_codes(x):
    """Blocks of 32: codes with element j in byte j's low half and element j + 16 in its high half, and f16 scales"""
    b = x.unflatten(-1, (-1, 32))
    hi, lo = b.amax(-1), b.amin(-1)
    d = (torch.where(hi >= -lo, hi, lo) / -8).clamp(-2720, 2720).bfloat16().half()
    d32 = d.float()[..., None]
    c = torch.where(d32 == 0, torch.full_like(b, 8), (b / d32 + 8.5).floor().clamp(0, 15)).to(torch.uint8)
    return (c[..., :16] | (c[..., 16:] << 4)).flatten(-2), d


def _values(codes, scales):
    b = codes.unflatten(-1, (-1, 16))
    c = torch.cat([b & 15, b >> 4], -1).float() - 8
    return (c * scales.float()[..., None]).flatten(-2)


def _append_plain(st):
    case = st["case"]
    H, Nkv, D, P = case["heads"], case["kv_heads"], case["dim"], case["page"]
    x = st["qkv"].float().view(-1, H + 2 * Nkv, D)
    q = _rotate(_norm(x[:, :H], st["q_norm"]), st["pos"], st["rope"], case["layout"])
    k = _rotate(_norm(x[:, H:H + Nkv], st["k_norm"]), st["pos"], st["rope"], case["layout"])
    page, off = st["table"][st["seq"].long(), (st["pos"] // P).long()].long(), (st["pos"] % P).long()
    for n, val in (("k", k), ("v", x[:, H + Nkv:])):
        codes, scales = _to_codes(val)
        st[n + "c"][page, :, off] = codes
        st[n + "s"][page, :, off] = scales
    back = [_values(st[n + "c"][page, :, off], st[n + "s"][page, :, off]).half() for n in ("k", "v")]
    return {"q": q.to(st["qkv"].dtype), "k": back[0], "v": back[1]}


def _attn_plain(st):
    case = st["case"]
    H, Nkv, D, P, n_seq = case["heads"], case["kv_heads"], case["dim"], case["page"], case["n_seq"]
    dev, Q, K = st["q"].device, st["max_q"], st["max_kv"]
    q_len = st["q_start"].diff()
    i = torch.arange(Q, device=dev)
    at = (st["q_start"][:-1, None] + i).clamp(max=st["q"].shape[0] - 1).long()
    q = st["q"][at].float().view(n_seq, Q, Nkv, H // Nkv, D).permute(0, 2, 3, 1, 4).reshape(n_seq, Nkv, -1, D)
    pages = st["table"][:, :-(-K // P)].clamp(min=0).long()
    kv = [_values(st[n + "c"][pages], st[n + "s"][pages]).permute(0, 2, 1, 3, 4).reshape(n_seq, Nkv, -1, D)[:, :, :K]
          for n in ("k", "v")]
    s = (q @ kv[0].transpose(-1, -2) * D ** -0.5).view(n_seq, Nkv, H // Nkv, Q, K)
    last = (st["kv_len"] - q_len)[:, None] + i
    j = torch.arange(K, device=dev)
    seen = (j <= last[..., None]) & (j < st["kv_len"][:, None, None])
    if case["window"]:
        seen &= j > last[..., None] - case["window"]
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    p = (s - s.amax(-1, keepdim=True).clamp(min=-1e30)).exp()
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    o = (p.view(n_seq, Nkv, -1, K) @ kv[1]).view(n_seq, Nkv, H // Nkv, Q, D).permute(0, 3, 1, 2, 4).reshape(n_seq, Q, H, D)
    return o[i < q_len[:, None]].to(st["q"].dtype)


def _logits_plain(st):
    x = st["x"].float()
    R, V = x.shape
    L = st["hist"].shape[1]
    j = torch.arange(L, device=x.device)
    inside, made = j < st["hist_len"][:, None], j >= st["prompt_len"][:, None]
    ids = st["hist"].long()
    zero = torch.zeros_like(x)
    seen = zero.scatter_add(1, ids, inside.float()) > 0
    count = zero.scatter_add(1, ids, (inside & made).float())
    r = st["rep"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - st["freq"][:, None] * count - torch.where(count > 0, st["pres"][:, None], zero)
    if "bias_ids" in st:
        b = st["bias_ids"].long()  # of entries with one id the last one holds
        n = torch.arange(1, b.shape[1] + 1, device=x.device).expand_as(b)
        last = torch.zeros((R, V), dtype=torch.long, device=x.device).scatter_reduce(1, b, n, "amax")
        bias = torch.cat([zero[:, :1], st["bias_val"]], 1).gather(1, last)
        x = torch.where(last > 0, x + bias, x)
    if "mask" in st:
        bits = st["mask"][st["mask_row"].clamp(min=0).long()]
        open_ = (bits[:, :, None] >> torch.arange(32, device=x.device) & 1).bool().view(R, -1)[:, :V]
        x = x.masked_fill(~open_ & (st["mask_row"] >= 0)[:, None], -math.inf)
    return x.to(st["out"].dtype)


def run(state):
    st, case = state, state["case"]
    op = case["op"]
    if op == "rope":
        if own:
            return _acb().rope(st["x"], st["pos"], st["rope"], layout=case["layout"], inverse=case["inverse"], out=st["out"])
        return _rotate(st["x"].float(), st["pos"], st["rope"], case["layout"], case["inverse"]).to(st["x"].dtype)
    if op == "append":
        if own:
            c = st["cache"]
            c.append(st["qkv"], case["heads"], st["seq"], st["pos"], st["rope"], layout=case["layout"], q_norm=st["q_norm"],
                     k_norm=st["k_norm"], eps=1e-6, q_out=st["out"])
            c.read(st["seq"], st["pos"], k_out=st["k_out"], v_out=st["v_out"])
            return {"q": st["out"], "k": st["k_out"], "v": st["v_out"]}
        return _append_plain(st)
    if op == "attn":
        if own:
            return st["cache"].attention(st["q"], st["kv_len"], q_start=st["q_start"], max_q_len=st["max_q"],
                                         max_kv_len=st["max_kv"], window=case["window"], out=st["out"], work=st["work"])
        return _attn_plain(st)
    if own:
        return _acb().logits_rules(st["x"], hist=st["hist"], hist_len=st["hist_len"], prompt_len=st["prompt_len"],
                                      rep=st["rep"], freq=st["freq"], pres=st["pres"], bias_ids=st.get("bias_ids"),
                                      bias_val=st.get("bias_val"), mask=st.get("mask"), mask_row=st.get("mask_row"),
                                      out=st["out"])
    return _logits_plain(st)


# ---- what a pass cannot do without --------------------------------------------------------------------

def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}
    op = case["op"]
    if op == "rope":
        n = case["n_tok"] * case["heads"]
        return {"bytes": 2 * n * case["dim"] * size[case["dtype"]] + case["n_tok"] * (4 + 4 * case["rope_dim"]),
                "flops": 3 * n * case["rope_dim"]}
    if op == "logits":
        R, V = case["rows"], case["vocab"]
        hist = sum(_spread(R, (case["hist"] + 1) // 2, case["hist"], 0.61803))
        b = R * V * (size[case["dtype"]] + size[case["out"]]) + 4 * hist + 8 * R * case["bias"] + 20 * R
        return {"bytes": b + min(case["masks"], (R + 1) // 2) * V // 8, "flops": 2 * R * V}
    H, Nkv, D, e = case["heads"], case["kv_heads"], case["dim"], size[case["dtype"]]
    q_len, kv_len = _lens(case)
    row = 2 * Nkv * (D // 2 + D // 32 * 2)  # a token's keys and values as codes and scales
    if op == "append":
        T = sum(q_len)
        # the rows of qkv, the rotated q, the rows of the cache, and these read back as f16
        return {"bytes": T * ((2 * H + 2 * Nkv) * D * e + 2 * row + 4 * Nkv * D + 4 * case["rope_dim"] + 8),
                "flops": T * (8 * H + 12 * Nkv) * D}
    byt, flops = 0, 0
    for n, m in zip(q_len, kv_len):
        first = max(0, m - n + 1 - case["window"]) if case["window"] else 0
        byt += 2 * n * H * D * e + (m - first) * row
        for i in range(n):
            last = m - n + i + 1
            flops += 4 * D * H * (min(last, case["window"]) if case["window"] else last)
    return {"bytes": byt, "flops": flops}


# ---- the definitions in 64 bits ------------------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "logits":
        out = torch.empty(st["x"].shape, dtype=torch.float64, device=st["x"].device)
        for r in range(case["rows"]):
            x = st["x"][r].double()
            h = st["hist"][r, :int(st["hist_len"][r])].long()
            ids = torch.unique(h)
            rep = st["rep"][r].double()
            x[ids] = torch.where(x[ids] > 0, x[ids] / rep, x[ids] * rep)
            ids, n = torch.unique(h[int(st["prompt_len"][r]):], return_counts=True)
            x[ids] -= st["freq"][r].double() * n + st["pres"][r].double()
            if case["bias"]:
                b = dict(zip(st["bias_ids"][r].tolist(), st["bias_val"][r].double().tolist()))
                x[torch.tensor(list(b), device=x.device)] += torch.tensor(list(b.values()), dtype=x.dtype, device=x.device)
            if case["masks"] and int(st["mask_row"][r]) >= 0:
                w = st["mask"][int(st["mask_row"][r])].cpu().numpy().view("u1")
                bits = torch.from_numpy(np.unpackbits(w, bitorder="little")[:case["vocab"]]).to(x.device)
                x[bits == 0] = -math.inf
            out[r] = x
        return out

    def turn(x, pos, inverse=False):
        R = st["rope"].shape[1]
        t = st["rope"][pos.long()].double()
        z = torch.complex(t[:, None, 0::2], t[:, None, 1::2])
        z = z.conj() if inverse else z
        y = x.clone()
        if case["layout"] == "half":
            w = torch.complex(x[..., :R // 2], x[..., R // 2:R]) * z
            y[..., :R // 2], y[..., R // 2:R] = w.real, w.imag
        else:
            w = torch.view_as_complex(x[..., :R].unflatten(-1, (-1, 2)).contiguous()) * z
            y[..., :R] = torch.view_as_real(w).flatten(-2)
        return y

    if op == "rope":
        return turn(st["x"].double(), st["pos"], case["inverse"])
    H, Nkv, D = case["heads"], case["kv_heads"], case["dim"]

    def held(x):
        b = x.reshape(*x.shape[:-1], -1, 32)
        far = b.abs().amax(-1, keepdim=True)  # its sign: positive where both signs have it
        d = (torch.where((b == far).any(-1, keepdim=True), far, -far) / -8).clamp(-2720, 2720).bfloat16().half().double()
        c = torch.where(d == 0, torch.full_like(b, 8.0), (b / d + 8.5).floor()).clamp(0, 15)
        return ((c - 8) * d).reshape(x.shape)

    if op == "append":
        x = st["qkv"].double().view(-1, H + 2 * Nkv, D)
        n = lambda y, w: y if w is None else y / (y.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()  # noqa: E731
        return {"q": turn(n(x[:, :H], st["q_norm"]), st["pos"]),
                "k": held(turn(n(x[:, H:H + Nkv], st["k_norm"]), st["pos"])), "v": held(x[:, H + Nkv:])}

    if work(case)["flops"] > 2e12:
        return None
    out = torch.empty(st["q"].shape, dtype=torch.float64, device=st["q"].device)
    start, G = st["q_start"].tolist(), H // Nkv
    for s, m in enumerate(st["kv_len"].tolist()):
        n = start[s + 1] - start[s]
        pages = st["table"][s, :-(-m // case["page"])].long()
        pos = torch.arange(m - n, m, device=out.device)[:, None]
        j = torch.arange(m, device=out.device)
        seen = (j <= pos) & ((j > pos - case["window"]) if case["window"] else True)
        for h in range(Nkv):
            k, v = (_unpacked(st[a + "c"][pages, h], st[a + "s"][pages, h])[:m] for a in "kv")
            for i in range(h * G, (h + 1) * G):
                z = st["q"][start[s]:start[s + 1], i].double() @ k.T / math.sqrt(D)
                out[start[s]:start[s + 1], i] = torch.softmax(z.masked_fill(~seen, -math.inf), -1) @ v
    return out


def _unpacked(codes, scales):
    """[pages, page, D/2] and [pages, page, D/32] -> [tokens, D] in 64 bits"""
    n, P, half = codes.shape
    b = codes.reshape(n * P, half // 16, 16).long()
    x = torch.empty((n * P, half // 16, 32), dtype=torch.float64, device=codes.device)
    x[..., :16], x[..., 16:] = b % 16 - 8, b // 16 - 8
    return (x * scales.reshape(n * P, half // 16, 1).double()).reshape(n * P, half * 2)
