"""Timed operators of a recurrent mixer layer: causal convolution, selective scan, gated norm, residual norm.

A batch is packed and ragged: sequence b's rows are rows starts[b] .. starts[b + 1] - 1 of every
tensor. What a sequence carries from one call to the next lies in a pool of states, slot
slots[b] of it; a sequence at position 0 (offsets[b]) starts from zeros.

Kinds (the ``kind`` field):

``conv``      short causal convolution of every channel over time, bias, SiLU. Outputs: the rows and
              the pool of each sequence's last width - 1 inputs.
``scan``      dt = softplus(raw + bias); h = exp(dt A) h + dt x B^T; y = h C + D x for every head, h of
              head_dim x d_state values. Outputs: y and the pool of states (32 bits).
``gated``     RMSNorm of groups of a row, gated by silu(gate) before or after the norm. Output: the rows.
``residual``  h = residual + scale * gate * norm(branch), out = norm(h): the norms after one block and
              before the next. Outputs: out and the residual stream.

``run`` computes them in plain torch, or with the framework's kernels where ``own`` is true;
``exact`` from the definitions in float64.
"""
import math
import os
import random
import sys

import torch
import torch.nn.functional as F

own = False

EPS = 1e-6
CHUNK = 64  # tokens of a chunk of the plain scan
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
# heads, head_dim, d_state, groups of B and C
SCANS = [(64, 64, 128, 8), (80, 64, 128, 1), (24, 64, 128, 1), (32, 64, 64, 2), (16, 128, 128, 2), (12, 48, 80, 3)]
# values of a row, values of a group of the norm
NORMS = [(4096, 128), (4096, 512), (4096, 4096), (5120, 5120), (2048, 256), (1000, 40)]
DIMS = [1024, 2048, 2560, 4096, 5120, 1111]


def listed():
    return [
        # One new token of one user, the q|k|v channels of 16 key and 32 value heads of 128.
        dict(name="conv_token_b1", kind="conv", type="bf16", batch=1, new=1, ragged=False, fresh=False, channels=8192,
             width=4, bias=False),
        # One new token for each of 64 users.
        dict(name="conv_step_b64", kind="conv", type="bf16", batch=64, new=1, ragged=False, fresh=False, channels=8192,
             width=4, bias=False),
        # Eight prompts of different lengths taken in together, channels of a state space layer.
        dict(name="conv_prompts_b8", kind="conv", type="bf16", batch=8, new=2048, ragged=True, fresh=True,
             channels=6144, width=4, bias=True),
        # The smallest scan: one new token of one user.
        dict(name="scan_token_b1", kind="scan", type="bf16", batch=1, new=1, ragged=False, fresh=False, heads=64,
             head_dim=64, d_state=128, groups=8),
        # A decode step of 32 users: the states decide.
        dict(name="scan_step_b32", kind="scan", type="bf16", batch=32, new=1, ragged=False, fresh=False, heads=64,
             head_dim=64, d_state=128, groups=8),
        # Four prompts of up to 2048 tokens from the start.
        dict(name="scan_prompts_b4_2k", kind="scan", type="bf16", batch=4, new=2048, ragged=True, fresh=True, heads=64,
             head_dim=64, d_state=128, groups=8),
        # The second 8192 tokens of one long document: few heads times sequences, time has to be split.
        dict(name="scan_chunk_b1_8k", kind="scan", type="bf16", batch=1, new=8192, ragged=False, fresh=False, heads=64,
             head_dim=64, d_state=128, groups=8),
        # Odd sizes in 32 bits, as a check of a small model's layer runs.
        dict(name="scan_odd_f32", kind="scan", type="f32", batch=3, new=301, ragged=True, fresh=False, heads=12,
             head_dim=48, d_state=80, groups=3),
        # The scan's output of 32 users: 32 heads of 128, each normed alone, then gated.
        dict(name="gated_step_b32", kind="gated", type="bf16", rows=32, dim=4096, group=128, first=False, shared=True),
        # The same for a long prompt of a state space layer: gated, then normed in groups of 512.
        dict(name="gated_8k", kind="gated", type="bf16", rows=8192, dim=4096, group=512, first=True, shared=False),
        # One token between two blocks.
        dict(name="residual_token", kind="residual", type="bf16", rows=1, dim=2048, post=False, gate="none",
             stream="bf16"),
        # A long prompt between two blocks: norms on both sides, a gate for each value, 32-bit residual stream.
        dict(name="residual_8k", kind="residual", type="bf16", rows=8192, dim=4096, post=True, gate="rows",
             stream="f32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    c = dict(kind=rng.choice(["conv", "scan", "scan", "gated", "residual"]))
    if c["kind"] in ("conv", "scan"):
        step = rng.random() < 0.4
        batch = _log(rng, 1, 64)
        new = rng.choice([1, 1, rng.randint(2, 6)]) if step else _log(rng, 8, min(8192, 8192 // batch))
        c.update(batch=batch, new=new, ragged=rng.random() < 0.6, fresh=rng.random() < 0.4)
    if c["kind"] == "conv":
        c.update(type=rng.choice(["bf16", "bf16", "f16", "f32"]), channels=rng.choice([8192, 6144, 4352, 1031]),
                 width=rng.choice([4, 4, 3, 2]), bias=rng.random() < 0.5)
    elif c["kind"] == "scan":
        heads, head_dim, d_state, groups = rng.choice(SCANS)
        c.update(type=rng.choice(["bf16", "bf16", "bf16", "f16", "f32"]), heads=heads, head_dim=head_dim,
                 d_state=d_state, groups=groups)
        if c["type"] != "bf16":  # prompts of the wider types are checks: short
            c["new"] = min(c["new"], 600)
    elif c["kind"] == "gated":
        dim, group = rng.choice(NORMS)
        c.update(type=rng.choice(["bf16", "bf16", "f16", "f32"]), rows=_log(rng, 1, 6000), dim=dim, group=group,
                 first=rng.random() < 0.5, shared=rng.random() < 0.5)
    else:
        c.update(type=rng.choice(["bf16", "bf16", "f16", "f32"]), rows=_log(rng, 1, 6000), dim=rng.choice(DIMS),
                 post=rng.random() < 0.5, gate=rng.choice(["none", "one", "rows"]),
                 stream="f32" if rng.random() < 0.5 else "same")
    return c


def _lengths(case):
    rng = random.Random("%(batch)d %(new)d %(kind)s" % case)
    new = [rng.randint(1, case["new"]) if case["ragged"] else case["new"] for _ in range(case["batch"])]
    if case["ragged"]:
        new[0] = case["new"]
    return new


def _randn(gen, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 6007 + 29)
    dtype = TYPES[case["type"]]
    s = dict(case=case)
    if case["kind"] in ("conv", "scan"):
        new, batch = _lengths(case), case["batch"]
        rows = sum(new)
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        n_slots = batch + 1  # one that no sequence of this call has
        s.update(
            starts=torch.tensor(starts, dtype=torch.int32, device="cuda") if case["ragged"] else None,
            offsets=torch.full((batch,), 0 if case["fresh"] else 1000, dtype=torch.int32, device="cuda"),
            slots=torch.randperm(n_slots, generator=gen, device="cuda")[:batch].to(torch.int32), max_rows=max(new),
            # of each packed row: its sequence, and its place among the sequence's rows
            row_b=torch.repeat_interleave(torch.arange(batch), torch.tensor(new)).cuda())
        s["row_t"] = torch.arange(rows, device="cuda") - torch.tensor(starts, device="cuda")[s["row_b"]]
        s["n"] = torch.tensor(new, device="cuda")
    if case["kind"] == "conv":
        C, W = case["channels"], case["width"]
        # the convolved channels are a part of the projection's rows
        s["x"] = _randn(gen, rows, C + 64, dtype=dtype)[:, 32:32 + C] if C % 8 == 0 else _randn(gen, rows, C, dtype=dtype)
        s["w"] = (_randn(gen, C, W) / math.sqrt(W)).to(dtype)
        s["bias"] = (0.1 * _randn(gen, C)).to(dtype) if case["bias"] else None
        s["state"] = _randn(gen, n_slots, W - 1, C, dtype=dtype)
        s["y"] = torch.empty(rows, C, dtype=dtype, device="cuda")
    elif case["kind"] == "scan":
        H, P, N, G = case["heads"], case["head_dim"], case["d_state"], case["groups"]
        # x, B and C are parts of the convolution's rows, dt of the projection's
        xbc = F.silu(_randn(gen, rows, H * P + 2 * G * N)).to(dtype)
        s["x"] = xbc[:, :H * P].unflatten(1, (H, P))
        s["B"] = xbc[:, H * P:H * P + G * N].unflatten(1, (G, N))
        s["C"] = xbc[:, H * P + G * N:].unflatten(1, (G, N))
        s["dt"] = _randn(gen, rows, H + 32, dtype=dtype)[:, 32:]
        s["A"] = -(1 + 15 * torch.rand(H, generator=gen, device="cuda"))
        dt0 = torch.exp(torch.rand(H, generator=gen, device="cuda") * math.log(100.0) + math.log(1e-3))
        s["dt_bias"] = dt0 + torch.log(-torch.expm1(-dt0))
        s["D"] = 1 + 0.1 * _randn(gen, H)
        s["state"] = 0.1 * _randn(gen, n_slots, H, P, N)  # the size that such inputs keep it at
        s["y"] = torch.empty(rows, H, P, dtype=dtype, device="cuda")
    elif case["kind"] == "gated":
        rows, dim = case["rows"], case["dim"]
        s["x"] = _randn(gen, rows, dim, dtype=dtype)
        s["gate"] = _randn(gen, rows, 2 * dim, dtype=dtype)[:, :dim]  # a part of the projection's rows
        s["w"] = (1 + 0.1 * _randn(gen, case["group"] if case["shared"] else dim)).to(dtype)
        s["y"] = torch.empty(rows, dim, dtype=dtype, device="cuda")
    else:
        rows, dim = case["rows"], case["dim"]
        s["branch"] = _randn(gen, rows, dim, dtype=dtype)
        s["residual"] = _randn(gen, rows, dim, dtype=torch.float32 if case["stream"] == "f32" else dtype)
        s["pre_w"] = (1 + 0.1 * _randn(gen, dim)).to(dtype)
        s["post_w"] = (1 + 0.1 * _randn(gen, dim)).to(dtype) if case["post"] else None
        s["gate"] = {"none": None, "one": _randn(gen, dim, dtype=dtype),
                     "rows": _randn(gen, rows, dim, dtype=dtype)}[case["gate"]]
        s["out"] = torch.empty(rows, dim, dtype=dtype, device="cuda")
    return s


SCALE = 0.5  # of the branch that joins the residual stream


def _plain_conv(s):
    W = s["case"]["width"]
    slots = s["slots"].long()
    # each sequence's kept inputs, then its rows, padded to the longest
    x = torch.zeros(len(slots), W - 1 + s["max_rows"], s["case"]["channels"], device="cuda")
    x[:, :W - 1] = torch.where((s["offsets"] > 0)[:, None, None], s["state"][slots].float(), 0.0)
    x[s["row_b"], W - 1 + s["row_t"]] = s["x"].float()
    tap = torch.arange(W, device="cuda")
    seen = x.unfold(1, W, 1)[s["row_b"], s["row_t"]]  # [rows, channels, W]
    y = (seen * s["w"].float()).sum(-1)
    if s["bias"] is not None:
        y = y + s["bias"].float()
    s["state"][slots] = x[torch.arange(len(slots), device="cuda")[:, None], s["n"][:, None] + tap[:W - 1]].to(s["x"].dtype)
    return {"y": (y * torch.sigmoid(y)).to(s["x"].dtype), "state": s["state"]}


def _plain_scan(s):
    c = s["case"]
    H, P, N, G = c["heads"], c["head_dim"], c["d_state"], c["groups"]
    B, Q = c["batch"], min(CHUNK, s["max_rows"])
    n_chunks = -(-s["max_rows"] // Q)
    slots = s["slots"].long()

    def padded(t):  # [B, chunks, Q, ...], zeros behind a sequence's rows
        out = torch.zeros(B, n_chunks * Q, *t.shape[1:], dtype=t.dtype, device="cuda")
        out[s["row_b"], s["row_t"]] = t
        return out.view(B, n_chunks, Q, *t.shape[1:])

    raw = s["dt"].float() + s["dt_bias"]
    dt = torch.where(raw > 20, raw, torch.log1p(torch.exp(raw.clamp(max=20))))
    x = padded(s["x"].float() * dt[..., None]).permute(0, 1, 3, 2, 4)  # [B, chunks, H, Q, P]
    Bm, Cm = (padded(s[k].float()).permute(0, 1, 3, 2, 4) for k in ("B", "C"))  # [B, chunks, G, Q, N]
    a = padded((dt * s["A"]).double()).permute(0, 1, 3, 2)  # [B, chunks, H, Q]
    upto = a.cumsum(-1)  # differences of long sums: 64 bits
    t = torch.arange(Q, device="cuda")
    decay = torch.exp((upto[..., :, None] - upto[..., None, :]).float().masked_fill(t[:, None] < t, -math.inf))
    scores = torch.matmul(Cm, Bm.transpose(-1, -2).contiguous())
    rep = H // G
    y = torch.matmul(scores.repeat_interleave(rep, 2) * decay, x)
    # what each chunk adds to the state at its end, and the state before each chunk
    to_end = torch.exp((upto[..., -1:] - upto).float())
    own_h = torch.matmul((x * to_end[..., None]).transpose(-1, -2).contiguous(), Bm.repeat_interleave(rep, 2))
    h0 = torch.where((s["offsets"] > 0)[:, None, None, None], s["state"][slots], 0.0)
    h = torch.cat([h0[:, None], own_h], 1).permute(0, 2, 1, 3, 4).reshape(B, H, n_chunks + 1, P * N)
    sums = F.pad(upto[..., -1].permute(0, 2, 1).cumsum(-1), (1, 0))  # [B, H, chunks + 1]
    k = torch.arange(n_chunks + 1, device="cuda")
    carry = torch.exp((sums[..., :, None] - sums[..., None, :]).float().masked_fill(k[:, None] < k, -math.inf))
    h = torch.matmul(carry, h).view(B, H, n_chunks + 1, P, N)
    before = h[:, :, :-1].transpose(1, 2)  # [B, chunks, H, P, N]
    y = y + torch.matmul(Cm.repeat_interleave(rep, 2), before.transpose(-1, -2).contiguous()) * torch.exp(upto).float()[..., None]
    y = y.permute(0, 1, 3, 2, 4).reshape(B, n_chunks * Q, H, P)[s["row_b"], s["row_t"]]
    s["state"][slots] = h[:, :, -1]
    return {"y": (y + s["D"][:, None] * s["x"].float()).to(s["x"].dtype), "state": s["state"]}


def _norm(x, w):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w


def _plain_gated(s):
    c = s["case"]
    x, z = (s[k].float().unflatten(1, (-1, c["group"])) for k in ("x", "gate"))
    w = s["w"].float().view(-1, c["group"])
    act = z * torch.sigmoid(z)
    y = _norm(x * act, w) if c["first"] else _norm(x, w) * act
    return y.flatten(1).to(s["x"].dtype)


def _plain_residual(s):
    u = s["branch"].float()
    if s["post_w"] is not None:
        u = _norm(u, s["post_w"].float())
    if s["gate"] is not None:
        u = u * s["gate"].float()
    h = s["residual"].float() + SCALE * u
    s["residual"].copy_(h)
    return {"out": _norm(h, s["pre_w"].float()).to(s["branch"].dtype), "residual": s["residual"]}


def _framework(s):
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "engine-mlx_amd")
    if here not in sys.path:
        sys.path.insert(0, here)
    import ema_attn as ema

    c = s["case"]
    s["ema"] = ema
    if c["kind"] == "scan":
        s["workspace"] = ema.ssm_workspace(c["batch"], s["x"].shape[0], s["max_rows"], c["heads"], c["head_dim"],
                                           c["d_state"], c["groups"], dtype=s["x"].dtype)


def run(s):
    c = s["case"]
    if own:
        if "ema" not in s:  # the workspace, kept by the program
            _framework(s)
        ema = s["ema"]
        if c["kind"] == "conv":
            ema.causal_conv(s["x"], s["w"], bias=s["bias"], state=s["state"], starts=s["starts"], offsets=s["offsets"],
                            slots=s["slots"], max_rows=s["max_rows"], out=s["y"])
            return {"y": s["y"], "state": s["state"]}
        if c["kind"] == "scan":
            ema.ssm_scan(s["x"], s["dt"], s["B"], s["C"], s["A"], s["state"], D=s["D"], dt_bias=s["dt_bias"],
                         starts=s["starts"], offsets=s["offsets"], slots=s["slots"], max_rows=s["max_rows"],
                         out=s["y"], workspace=s["workspace"])
            return {"y": s["y"], "state": s["state"]}
        if c["kind"] == "gated":
            return ema.gated_norm(s["x"], s["gate"], s["w"], EPS, group=c["group"], gate_first=c["first"], out=s["y"])
        ema.residual_norm(s["branch"], s["residual"], s["pre_w"], EPS, post_weight=s["post_w"], gate=s["gate"],
                          scale=SCALE, out=s["out"])
        return {"out": s["out"], "residual": s["residual"]}
    return {"conv": _plain_conv, "scan": _plain_scan, "gated": _plain_gated, "residual": _plain_residual}[c["kind"]](s)


def work(case):
    size = 4 if case["type"] == "f32" else 2
    if case["kind"] == "conv":  # rows in and out, the kept inputs in (past a start) and out, taps and bias
        rows, C, W = sum(_lengths(case)), case["channels"], case["width"]
        kept = case["batch"] * (W - 1) * C * (1 if case["fresh"] else 2)
        return {"bytes": (2 * rows * C + kept + C * (W + case["bias"])) * size, "flops": rows * C * (2 * W + 4)}
    if case["kind"] == "scan":
        H, P, N, G = case["heads"], case["head_dim"], case["d_state"], case["groups"]
        new = _lengths(case)
        rows = sum(new)
        states = case["batch"] * H * P * N * 4 * (1 if case["fresh"] else 2)
        # h = a h + x B^T and y = h C for every token
        return {"bytes": rows * (2 * H * P + H + 2 * G * N) * size + states + 3 * H * 4, "flops": rows * H * P * N * 5}
    rows, dim = case["rows"], case["dim"]
    if case["kind"] == "gated":
        return {"bytes": (3 * rows * dim + (case["group"] if case["shared"] else dim)) * size, "flops": rows * dim * 10}
    gate = {"none": 0, "one": dim, "rows": rows * dim}[case["gate"]]
    stream = 4 if case["stream"] == "f32" else size
    return {"bytes": (2 * rows * dim + gate + dim * (1 + case["post"])) * size + 2 * rows * dim * stream,
            "flops": rows * dim * 10}


def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    if case["kind"] == "gated":
        x, z = s["x"].to(f64), s["gate"].to(f64)
        act = z / (1 + torch.exp(-z))
        if case["first"]:
            x = x * act
        y = torch.empty_like(x)
        for i in range(0, case["dim"], case["group"]):
            part = slice(i, i + case["group"])
            w = s["w"] if case["shared"] else s["w"][part]
            y[:, part] = x[:, part] / torch.sqrt(x[:, part].pow(2).sum(1, keepdim=True) / case["group"] + EPS) * w.to(f64)
        return y if case["first"] else y * act
    if case["kind"] == "residual":
        u, dim = s["branch"].to(f64), case["dim"]
        if case["post"]:
            u = u / torch.sqrt((u * u).sum(1, keepdim=True) / dim + EPS) * s["post_w"].to(f64)
        if s["gate"] is not None:
            u = u * s["gate"].to(f64)
        h = s["residual"].to(f64) + u * SCALE
        return {"out": h / torch.sqrt((h * h).sum(1, keepdim=True) / dim + EPS) * s["pre_w"].to(f64), "residual": h}
    new = _lengths(case)
    state = s["state"].to(f64)
    at = 0
    if case["kind"] == "conv":
        W = case["width"]
        y = torch.empty(sum(new), case["channels"], dtype=f64, device="cuda")
        for b, n in enumerate(new):
            slot = int(s["slots"][b])
            x = torch.cat([state[slot] * (0 if case["fresh"] else 1), s["x"][at:at + n].to(f64)])
            z = sum(x[j:j + n] * s["w"][:, j].to(f64) for j in range(W))
            z = z if s["bias"] is None else z + s["bias"].to(f64)
            y[at:at + n] = z / (1 + torch.exp(-z))
            state[slot] = x[n:]
            at += n
        return {"y": y, "state": state}
    H, G = case["heads"], case["groups"]
    group = torch.arange(H, device="cuda") // (H // G)
    dt = F.softplus(s["dt"].to(f64) + s["dt_bias"].to(f64), threshold=50)
    a = torch.exp(dt * s["A"].to(f64))
    y = torch.empty(s["x"].shape, dtype=f64, device="cuda")
    # token by token, all sequences that have one
    starts = [sum(new[:b]) for b in range(len(new))]
    slots = s["slots"].long()
    h = state[slots] * (0 if case["fresh"] else 1)
    for t in range(max(new)):
        on = [b for b in range(len(new)) if new[b] > t]
        r = [starts[b] + t for b in on]
        x, Bm, Cm = s["x"][r].to(f64), s["B"][r].to(f64)[:, group], s["C"][r].to(f64)[:, group]
        whole = len(on) == len(new)
        g = h if whole else h[on]
        g = g * a[r][..., None, None] + (dt[r][..., None] * x)[..., None] * Bm[:, :, None]
        y[r] = (g * Cm[:, :, None]).sum(-1) + s["D"].to(f64)[:, None] * x
        if whole:
            h = g
        else:
            h[on] = g
    state[slots] = h
    return {"y": y, "state": state}
