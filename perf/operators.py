"""Timed operators of the paged KV cache: append, attention over pages, attention over a shared prefix.

A paged cache keeps K and V in pages of ``page`` positions, [n_pages, n_kv, page, head_dim];
row b of ``table`` names the pages of sequence b in order (position p lies in slot p % page of
page table[b, p // page]). A batch is ragged: sequence b's query rows are rows
starts[b] .. starts[b + 1] - 1 of one packed tensor, and they are its newest positions.

Kinds (the ``kind`` field):

``append``   per head RMSNorm of q and k, split-half rotation at the row's position, k and v
             written to their slots. Outputs: q, the K pages, the V pages.
``attend``   causal attention of the rows over their sequence's pages (K/V rows in bf16, or
             E4M3 codes with one power-of-two scale per 64 values). Output: the rows.
``prefix``   the same where every sequence's own pages continue one shared prefix, held once.

``run`` computes them in plain torch, or with the framework's kernels where ``own`` is true;
``exact`` from the definitions in float64.
"""
import math
import os
import random
import sys

import torch

own = False

EPS, THETA = 1e-6, 1e6
D = 128
FP8_SCALE_DIMS = 64  # values of a row that share one scale
# query heads, kv heads: the layers of the 1.7B-, 8B- and 14B-size models, and one, two and
# four kv heads with groups of 12, 8 and 1
HEADS = [(16, 8), (32, 8), (40, 8), (12, 1), (16, 2), (4, 4)]
PAGES = [16, 32, 64, 128, 256]


def listed():
    return [
        # One new token of one user, 1.7B-size layer: the smallest call there is.
        dict(name="append_token_b1", kind="append", batch=1, new=1, ragged=False, past=1024, n_heads=16, n_kv=8,
             page=16),
        # One new token for each of 32 users of an 8B-size model.
        dict(name="append_step_b32", kind="append", batch=32, new=1, ragged=False, past=2000, n_heads=32, n_kv=8,
             page=64),
        # Eight prompts of different lengths taken in together, page ends inside the prompts.
        dict(name="append_prompts_b8", kind="append", batch=8, new=2048, ragged=True, past=0, n_heads=32, n_kv=8,
             page=16),
        # One user, 1000 tokens into a conversation, small pages: latency decides.
        dict(name="token_b1_1k", kind="attend", batch=1, new=1, ragged=False, past_min=1000, past=1000, n_heads=16,
             n_kv=8, page=16, pages="bf16"),
        # A decode step of 32 users, 512 to 8191 tokens each, 8B-size layer.
        dict(name="step_b32_8k", kind="attend", batch=32, new=1, ragged=False, past_min=511, past=8190, n_heads=32,
             n_kv=8, page=64, pages="bf16"),
        # The same step over pages held in FP8.
        dict(name="step_b32_8k_fp8", kind="attend", batch=32, new=1, ragged=False, past_min=511, past=8190,
             n_heads=32, n_kv=8, page=64, pages="fp8"),
        # Long documents: 8 users of 30000 to 32767 tokens. The most bytes.
        dict(name="step_b8_32k", kind="attend", batch=8, new=1, ragged=False, past_min=29999, past=32766, n_heads=32,
             n_kv=8, page=128, pages="bf16"),
        # Up to five drafted tokens of each of 16 users, checked in one pass, 14B-size layer.
        dict(name="drafts_b16_4k", kind="attend", batch=16, new=5, ragged=True, past_min=100, past=4000, n_heads=40,
             n_kv=8, page=32, pages="bf16"),
        # Four prompts of up to 2048 tokens from the start: matrix work decides.
        dict(name="prompts_b4_2k", kind="attend", batch=4, new=2048, ragged=True, past_min=0, past=0, n_heads=32,
             n_kv=8, page=16, pages="bf16"),
        # Four users on one 1500-token system prompt, a few own tokens each.
        dict(name="prefix_b4_1k5", kind="prefix", batch=4, new=1, ragged=False, prefix=1500, past_min=1, past=90,
             n_heads=32, n_kv=8, page=64),
        # 24 samples drawn from one 8000-token prompt, odd sizes.
        dict(name="prefix_b24_8k", kind="prefix", batch=24, new=1, ragged=False, prefix=8001, past_min=1, past=513,
             n_heads=40, n_kv=8, page=16),
        # 64 questions on one 32768-token document.
        dict(name="prefix_b64_32k", kind="prefix", batch=64, new=1, ragged=False, prefix=32768, past_min=20, past=400,
             n_heads=32, n_kv=8, page=128),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    n_heads, n_kv = rng.choice(HEADS)
    c = dict(kind=rng.choice(["append", "attend", "attend", "prefix"]), n_heads=n_heads, n_kv=n_kv,
             page=rng.choice(PAGES))
    if c["kind"] == "append":
        batch = _log(rng, 1, 64)
        new = _log(rng, 1, max(1, min(2048, 8000 // batch)))
        # positions up to 100000 for one user; fewer for many (the pages are held in whole)
        past = rng.choice([0, _log(rng, 1, 100000 // batch)])
        c.update(batch=batch, new=new, ragged=rng.random() < 0.7, past=past)
    elif c["kind"] == "attend":
        new = rng.choice([1, 1, rng.randint(2, 8), _log(rng, 16, 2048)])
        if new <= 8:
            batch = _log(rng, 1, 64)
            past = _log(rng, 1, min(32000, 160000 // batch))
        else:
            batch = _log(rng, 1, max(1, min(16, 6000 // new)))
            past = rng.choice([0, _log(rng, 1, max(1, min(16000, 5000000 // (batch * new))))])
        c.update(batch=batch, new=new, ragged=rng.random() < 0.7, past_min=min(past, rng.choice([0, past // 2, past])),
                 past=past, pages=rng.choice(["bf16", "fp8"]) if new <= 8 else "bf16")
    else:
        batch = _log(rng, 2, 64)
        past = _log(rng, 1, 1000)
        c.update(batch=batch, new=rng.choice([1, 1, 1, rng.randint(2, 4 if batch <= 16 else 2)]),
                 ragged=rng.random() < 0.5, prefix=_log(rng, 64, 32000 if batch <= 48 else 16000),
                 past_min=rng.randint(0, past), past=past)
        if c["new"] > 1:
            c["prefix"] = max(64, c["prefix"] // c["new"])
    return c


def _lengths(case):
    """Per sequence: new rows, and positions held before them (its own, behind a prefix)."""
    rng = random.Random("%(batch)d %(new)d %(past)d %(n_heads)d %(page)d" % case)
    new = [rng.randint(1, case["new"]) if case["ragged"] else case["new"] for _ in range(case["batch"])]
    past = [rng.randint(case.get("past_min", 0), case["past"]) for _ in range(case["batch"])]
    if case["ragged"]:
        new[0] = case["new"]
    past[-1] = case["past"]
    return new, past


def _table(counts, gen, spare=3):
    """Page numbers for sequences of counts[b] pages, in a shuffled order, -1 where there is no
    page; and how many pages there are."""
    total = sum(counts) + spare
    order = torch.randperm(total, generator=gen, device="cuda", dtype=torch.int64).to(torch.int32)
    table = torch.full((len(counts), max(max(counts), 1)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = order[at:at + n]
        at += n
    return table, total


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(torch.bfloat16)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 7919 + 17)
    new, past = _lengths(case)
    Hq, Hkv, P, B = case["n_heads"], case["n_kv"], case["page"], case["batch"]
    rows = sum(new)
    kv = [n + p for n, p in zip(new, past)]
    table, n_pages = _table([-(-n // P) for n in kv], gen)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    row_b = torch.repeat_interleave(torch.arange(B), torch.tensor(new)).cuda()
    s = dict(case=case, table=table, offsets=torch.tensor(past, dtype=torch.int32, device="cuda"),
             lengths=torch.tensor(kv, dtype=torch.int32, device="cuda"), max_len=max(kv), max_new=max(new),
             starts=torch.tensor(starts, dtype=torch.int32, device="cuda") if case["ragged"] else None,
             # of each packed row: its sequence, and its place among the sequence's rows
             row_b=row_b, row_t=torch.arange(rows, device="cuda") - torch.tensor(starts, device="cuda")[row_b])
    if case["kind"] == "append":
        s["qkv"] = _normal(gen, rows, (Hq + 2 * Hkv) * D)
        s["q_w"], s["k_w"] = ((1 + 0.1 * torch.randn(D, generator=gen, device="cuda")).to(torch.bfloat16)
                              for _ in range(2))
        s["k"], s["v"] = _normal(gen, n_pages, Hkv, P, D), _normal(gen, n_pages, Hkv, P, D)
        s["q"] = torch.empty(rows, Hq, D, dtype=torch.bfloat16, device="cuda")
        return s
    s["q"] = _normal(gen, rows, Hq, D)
    s["out"] = torch.empty(rows, Hq * D, dtype=torch.bfloat16, device="cuda")
    if case["kind"] == "prefix":
        n = -(-case["prefix"] // P)
        both = torch.randperm(n_pages + n, generator=gen, device="cuda").to(torch.int32)
        s["table"] = torch.where(table >= 0, both[table.clamp(min=0).long()], table)
        s["prefix_table"] = both[n_pages:].contiguous()
        s["prefix_len"] = torch.tensor([case["prefix"]], dtype=torch.int32, device="cuda")
        n_pages += n
    s["k"], s["v"] = _normal(gen, n_pages, Hkv, P, D), _normal(gen, n_pages, Hkv, P, D)
    if case.get("pages") == "fp8":
        for name in ("k", "v"):
            x = s[name].float().view(n_pages, Hkv, P, D // FP8_SCALE_DIMS, FP8_SCALE_DIMS)
            e = torch.ceil(torch.log2(x.abs().amax(-1, keepdim=True) / 448.0))
            s[name] = (x / torch.exp2(e)).to(torch.float8_e4m3fn).view(torch.uint8).view(n_pages, Hkv, P, D)
            s[name + "_exp"] = e.squeeze(-1).to(torch.int8)
    return s


def _rotate(x, angle):
    """Split-half rotation of x [rows, heads, D] (32 bits) by angle [rows, D / 2] (64 bits)."""
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    a, b = x[..., :D // 2], x[..., D // 2:]
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)


def _plain_append(s):
    Hq, Hkv, P = s["case"]["n_heads"], s["case"]["n_kv"], s["case"]["page"]
    x = s["qkv"].float().view(-1, Hq + 2 * Hkv, D)
    pos = s["offsets"].long()[s["row_b"]] + s["row_t"]
    angle = pos.double()[:, None] * THETA ** (-torch.arange(D // 2, device="cuda", dtype=torch.float64) / (D // 2))
    qk = x[:, :Hq + Hkv]
    qk = qk * torch.rsqrt(qk.square().mean(-1, keepdim=True) + EPS)
    q, k = _rotate(qk[:, :Hq] * s["q_w"].float(), angle), _rotate(qk[:, Hq:] * s["k_w"].float(), angle)
    page = s["table"].long()[s["row_b"], pos // P]
    s["k"][page, :, pos % P] = k.to(torch.bfloat16)
    s["v"][page, :, pos % P] = x[:, Hq + Hkv:].to(torch.bfloat16)
    return {"q": q.to(torch.bfloat16), "k": s["k"], "v": s["v"]}


def _gather(s, name, table):
    """The rows of the pages in table [.., n], in 32 bits: [.., n * page, n_kv, D]; zeros where
    there is no page."""
    x = s[name][table.clamp(min=0).long()]
    if s["case"].get("pages") == "fp8":
        e = s[name + "_exp"][table.clamp(min=0).long()].float()
        x = x.view(torch.float8_e4m3fn).float().unflatten(-1, (-1, FP8_SCALE_DIMS)) * torch.exp2(e)[..., None]
        x = x.flatten(-2)
    x = torch.where((table >= 0)[..., None, None, None], x.float(), 0.0)
    return x.transpose(-3, -2).flatten(-4, -3)


def _plain_attend(s):
    c = s["case"]
    Hq, Hkv, B, T = c["n_heads"], c["n_kv"], c["batch"], s["max_new"]
    G = Hq // Hkv
    # the packed rows padded to [B, Hkv, G * T, D]
    q = torch.zeros(B, T, Hq, D, device="cuda")
    q[s["row_b"], s["row_t"]] = s["q"].float()
    q = q.view(B, T, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * T, D)
    k = _gather(s, "k", s["table"])[:, :s["max_len"]].permute(0, 2, 3, 1)
    v = _gather(s, "v", s["table"])[:, :s["max_len"]].transpose(1, 2)
    scores = torch.matmul(q, k.contiguous()) * D ** -0.5
    key = torch.arange(s["max_len"], device="cuda")
    first = s["lengths"].long() - torch.bincount(s["row_b"], minlength=B)  # position of a sequence's first row
    last = first[:, None] + torch.arange(T, device="cuda")  # last key each row sees
    hidden = (key > last[..., None])[:, None, None]  # [B, 1, 1, T, L]
    scores = scores.view(B, Hkv, G, T, -1).masked_fill_(hidden, -math.inf).view(B, Hkv, G * T, -1)
    if c["kind"] == "prefix":
        pk = _gather(s, "k", s["prefix_table"])[:c["prefix"]].permute(1, 2, 0)
        pv = _gather(s, "v", s["prefix_table"])[:c["prefix"]].transpose(0, 1)
        rows = q.transpose(0, 1).reshape(Hkv, B * G * T, D)
        shared = torch.matmul(rows, pk.contiguous()).view(Hkv, B, G * T, -1).transpose(0, 1) * D ** -0.5
        p = torch.softmax(torch.cat([shared, scores], -1), -1)
        out = torch.matmul(p[..., c["prefix"]:], v.contiguous())
        p = p[..., :c["prefix"]].transpose(0, 1).reshape(Hkv, B * G * T, -1)
        out = out + torch.matmul(p, pv.contiguous()).view(Hkv, B, G * T, D).transpose(0, 1)
    else:
        out = torch.matmul(torch.softmax(scores, -1), v.contiguous())
    out = out.view(B, Hkv, G, T, D).permute(0, 3, 1, 2, 4).reshape(B, T, Hq * D)
    return out[s["row_b"], s["row_t"]].to(torch.bfloat16)


def _framework(s):
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "engine-mlx_amd")
    if here not in sys.path:
        sys.path.insert(0, here)
    import ema_attn as ema

    c = s["case"]
    Hq, Hkv, B = c["n_heads"], c["n_kv"], c["batch"]
    s["ema"] = ema
    s["cache"] = ema.PagedCache(s["k"].shape[0], Hkv, c["page"], D, k=s["k"], v=s["v"], dtype=c.get("pages", "bf16"),
                                k_exp=s.get("k_exp"), v_exp=s.get("v_exp"))
    if c["kind"] == "attend":
        s["workspace"] = ema.paged_workspace(B, s["q"].shape[0], Hq, Hkv, D, s["max_new"], s["max_len"])
    elif c["kind"] == "prefix":
        s["workspace"] = ema.paged_workspace(B, s["q"].shape[0], Hq, Hkv, D, s["max_new"], s["max_len"],
                                             max_prefix=c["prefix"])


def run(s):
    c = s["case"]
    if own:
        if "ema" not in s:  # the cache's handle and the workspace, kept by the program
            _framework(s)
        ema = s["ema"]
        if c["kind"] == "append":
            ema.paged_append(s["qkv"], s["q_w"], s["k_w"], EPS, THETA, s["offsets"], c["n_heads"], s["cache"],
                             s["table"], q_starts=s["starts"], q_out=s["q"])
            return {"q": s["q"], "k": s["k"], "v": s["v"]}
        if c["kind"] == "attend":
            return ema.paged_attention(s["q"], s["cache"], s["table"], s["lengths"], s["max_len"],
                                       q_starts=s["starts"], max_q=s["max_new"], out=s["out"],
                                       workspace=s["workspace"])
        return ema.prefix_attention(s["q"], s["cache"], s["prefix_table"], s["prefix_len"], c["prefix"], s["table"],
                                    s["lengths"], s["max_len"], q_starts=s["starts"], max_q=s["max_new"],
                                    out=s["out"], workspace=s["workspace"])
    return _plain_append(s) if c["kind"] == "append" else _plain_attend(s)


def work(case):
    new, past = _lengths(case)
    Hq, Hkv = case["n_heads"], case["n_kv"]
    rows, kv_row = sum(new), 2 * Hkv * D * 2
    if case["kind"] == "append":  # qkv in; q, k and v out; the norm weights
        return {"bytes": 2 * rows * (Hq + 2 * Hkv) * D * 2 + 4 * D, "flops": rows * (Hq + Hkv) * D * 8}
    if case.get("pages") == "fp8":  # codes, and a scale per 64 of them
        kv_row = 2 * Hkv * (D + D // FP8_SCALE_DIMS)
    # q in, the attended rows out, every K and V row that some query row sees, once
    held = sum(n + p for n, p in zip(new, past))
    pairs = sum(n * p + n * (n + 1) // 2 for n, p in zip(new, past))
    if case["kind"] == "prefix":
        held += case["prefix"]
        pairs += rows * case["prefix"]
    return {"bytes": 2 * rows * Hq * D * 2 + held * kv_row, "flops": 4 * D * Hq * pairs}


def exact(case, seed):
    s = prepare(case, seed)
    new, past = _lengths(case)
    Hq, Hkv, P = case["n_heads"], case["n_kv"], case["page"]
    G = Hq // Hkv
    f64 = torch.float64
    at = 0
    if case["kind"] == "append":
        k_pages, v_pages = s["k"].to(f64), s["v"].to(f64)
        q_out = torch.empty(sum(new), Hq, D, dtype=f64, device="cuda")
        freq = torch.exp(torch.arange(D // 2, dtype=f64, device="cuda") * (-2.0 * math.log(THETA) / D))
        for b, (n, p) in enumerate(zip(new, past)):
            x = s["qkv"][at:at + n].to(f64).view(n, Hq + 2 * Hkv, D)
            turn = torch.polar(torch.ones((), dtype=f64, device="cuda"),
                               torch.arange(p, p + n, dtype=f64, device="cuda")[:, None] * freq)[:, None]

            def head(x, w):
                y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / D + EPS) * w.to(f64)
                z = torch.complex(y[..., :D // 2], y[..., D // 2:]) * turn
                return torch.cat([z.real, z.imag], -1)

            q_out[at:at + n] = head(x[:, :Hq], s["q_w"])
            k, v = head(x[:, Hq:Hq + Hkv], s["k_w"]), x[:, Hq + Hkv:]
            for page in range(p // P, (p + n - 1) // P + 1):
                lo, hi = max(page * P, p), min(page * P + P, p + n)
                slot = slice(lo - page * P, hi - page * P)
                to = int(s["table"][b, page])
                k_pages[to, :, slot] = k[lo - p:hi - p].transpose(0, 1)
                v_pages[to, :, slot] = v[lo - p:hi - p].transpose(0, 1)
            at += n
        return {"q": q_out, "k": k_pages, "v": v_pages}

    def rows_of(name, pages, n):
        """[n_kv, n, D] of the first n positions held in the listed pages."""
        x = s[name][pages.long()]
        if case.get("pages") == "fp8":
            e = s[name + "_exp"][pages.long()].to(f64)
            x = x.view(torch.float8_e4m3fn).to(f64) * (2.0 ** e).repeat_interleave(FP8_SCALE_DIMS, -1)
        return x.to(f64).transpose(0, 1).reshape(Hkv, -1, D)[:, :n]

    out = torch.empty(sum(new), Hq, D, dtype=f64, device="cuda")
    prefix = case.get("prefix", 0)
    if prefix:
        shared = [rows_of(name, s["prefix_table"], prefix) for name in ("k", "v")]
    for b, (n, p) in enumerate(zip(new, past)):
        pages = s["table"][b, :-(-(n + p) // P)]
        k, v = (rows_of(name, pages, n + p) for name in ("k", "v"))
        if prefix:
            k, v = torch.cat([shared[0], k], 1), torch.cat([shared[1], v], 1)
        late = torch.arange(prefix + n + p, device="cuda") > torch.arange(n, device="cuda")[:, None] + (prefix + p)
        for h in range(Hq):
            e = s["q"][at:at + n, h].to(f64) @ k[h // G].T.contiguous() / math.sqrt(D)
            e = torch.exp(e.masked_fill(late, -math.inf) - e.masked_fill(late, -math.inf).amax(-1, keepdim=True))
            out[at:at + n, h] = (e / e.sum(-1, keepdim=True)) @ v[h // G]
        at += n
    return out.view(-1, Hq * D)
