"""Paged cache on the GPU against plain float64 (tests/paged_ref.py): append, attention over pages
and over a shared prefix. Slots that hold nothing are NaN throughout."""
import numpy as np
import pytest

import paged_ref as ref
from gpu_util import say

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ema():
    import torch

    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a ROCm GPU")
    import ema_attn

    ema_attn.lib()
    return ema_attn


def up(x, dtype=None):
    import torch

    t = torch.from_numpy(np.ascontiguousarray(x))
    return t.to(torch.bfloat16).cuda() if t.dtype == torch.float64 else t.cuda()


def down(t):
    return t.float().cpu().numpy().astype(np.float64)


def fp8_pool(x):
    """NaN-padded float64 pool -> (codes, exponents, the values they stand for); NaN rows get the
    NaN code 0x7F and exponent 127."""
    import torch

    nan = np.isnan(x).any(-1)
    y = np.where(nan[..., None], 0.0, x)
    blocks = y.reshape(x.shape[:-1] + (-1, 64))
    e = np.ceil(np.log2(np.maximum(np.abs(blocks).max(-1), 1e-4) / 448.0)).astype(np.int8)
    codes = torch.from_numpy(blocks / 2.0 ** e[..., None].astype(np.float64)).to(torch.float32).to(torch.float8_e4m3fn)
    val = codes.to(torch.float64).numpy() * 2.0 ** e[..., None].astype(np.float64)
    c = codes.view(torch.uint8).numpy().reshape(x.shape).copy()
    c[nan], e[nan] = 0x7F, 127
    return c, e, val.reshape(x.shape)


class OnGpu:
    """A ref.Batch on the device. order "nphd": pages as [page, position, head, D] in memory."""

    def __init__(self, ema, batch, pages="bf16", order="nhpd"):
        self.ema, self.b = ema, batch
        if pages == "fp8":
            (kc, ke, kv), (vc, ve, vv) = fp8_pool(batch.k), fp8_pool(batch.v)
            self.cache = ema.PagedCache(batch.n_pages, batch.Hkv, batch.page, batch.D, k=up(kc), v=up(vc), dtype="fp8",
                                        k_exp=up(ke), v_exp=up(ve))
            for held, table in [(h, t) for h, t in zip(batch.held, batch.table)] + [(batch.shared, batch.prefix_table)]:
                for x, val in ((held[0], kv), (held[1], vv)):
                    for p in range(-(-x.shape[0] // batch.page)):
                        n = min(batch.page, x.shape[0] - p * batch.page)
                        if 0 <= table[p] < batch.n_pages:
                            x[p * batch.page:p * batch.page + n] = val[table[p], :, :n].transpose(1, 0, 2)
        else:
            k, v = up(batch.k), up(batch.v)
            if order == "nphd":
                k, v = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v))
            self.cache = ema.PagedCache(batch.n_pages, batch.Hkv, batch.page, batch.D, k=k, v=v)
        self.table, self.starts = up(batch.table), up(batch.starts)
        self.lengths, self.q = up(np.asarray(batch.kv, np.int32)), up(batch.q)
        if batch.prefix:
            self.prefix_table, self.prefix_len = up(batch.prefix_table), up(np.asarray([batch.prefix], np.int32))

    def attention(self, **kw):
        b = self.b
        kw = dict(dict(q_starts=self.starts, max_q=max(b.new)), **kw)
        if b.prefix:
            return self.ema.prefix_attention(self.q, self.cache, self.prefix_table, self.prefix_len, b.prefix,
                                             self.table, self.lengths, max(b.kv), **kw)
        return self.ema.paged_attention(self.q, self.cache, self.table, self.lengths, max(b.kv), **kw)


def run(ema, batch, what, pages="bf16", order="nhpd", causal=True, scale=None, **kw):
    import torch

    say(f"{what}: new {batch.new[:8]} kv {batch.kv[:8]} page {batch.page} {batch.Hq}q/{batch.Hkv}kv")
    g = OnGpu(ema, batch, pages, order)
    if not batch.prefix:
        kw["causal"] = causal
    out = g.attention(scale=scale, **kw)
    torch.cuda.synchronize()
    want, mag = batch.attention(scale, causal)
    ref.check_attention(down(out), want, mag, what)
    return g, out


# ------------------------------------------------------------------ attention
LENGTHS = [
    ([1], [1]), ([1], [16]), ([1], [17]), ([1], [33]), ([1], [1000]),
    ([1] * 5, [1, 31, 32, 33, 257]),
    ([1, 0, 1, 1], [5, 40, 0, 64]),          # a sequence without rows, one that holds nothing
    ([0, 0, 3, 0], [0, 9, 7, 0]),
    ([5, 1, 3, 2], [70, 300, 3, 2]),         # drafted tokens; prompts as short as that
    ([4], [2]),                              # more rows than positions: the first two see nothing
    ([33, 1, 130], [33, 1, 400]),            # prompts, chunks and a single token in one call
    ([64, 65], [64, 65]),
]


@pytest.mark.parametrize("heads", [(4, 4), (16, 8), (10, 2), (12, 1), (16, 1)])
@pytest.mark.parametrize("new,kv", LENGTHS)
def test_attention_lengths(ema, new, kv, heads):
    for page in (16, 64):
        run(ema, ref.Batch(new, kv, page, *heads, seed=len(new) + sum(kv)), "paged attention")


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 2048])
@pytest.mark.parametrize("order", ["nhpd", "nphd"])
def test_attention_pages_and_orders(ema, page, order):
    run(ema, ref.Batch([1, 3, 1, 40], [700, 513, 15, 257], page, 8, 2, seed=page), f"page {page} {order}", order=order)


@pytest.mark.parametrize("new,kv", [([1] * 4, [1, 16, 333, 2050]), ([5, 2], [64, 1025]), ([150], [150])])
@pytest.mark.parametrize("page", [16, 64])
def test_attention_fp8(ema, new, kv, page):
    run(ema, ref.Batch(new, kv, page, 16, 4, seed=7), "fp8 pages", pages="fp8")


def test_attention_not_causal(ema):
    """An encoder's states: every row sees all of them, whatever the two lengths."""
    for new, kv in (([1, 7], [1500, 3]), ([130, 2], [40, 300]), ([3], [0])):
        run(ema, ref.Batch(new, kv, 32, 8, 4, seed=11), "not causal", causal=False)


@pytest.mark.parametrize("scale", [0.01, 1.0])
def test_attention_scales(ema, scale):
    run(ema, ref.Batch([1, 20], [900, 200], 16, 8, 2, seed=12), f"scale {scale}", scale=scale)


def test_attention_bad_pages(ema):
    """Entries outside the pool are not followed: their positions are zero rows."""
    holes = [(0, 0), (0, 3), (1, 2), (2, 0)]
    for pages in ("bf16", "fp8"):
        run(ema, ref.Batch([1, 40, 1], [100, 60, 10], 16, 8, 2, seed=13, holes=holes), "bad pages", pages=pages)


@pytest.mark.parametrize("B", [64, 65, 130, 1024])
def test_attention_many_sequences(ema, B):
    rng = np.random.default_rng(B)
    new, kv = rng.integers(0, 3, B), rng.integers(0, 70, B)
    new[0] = 1
    run(ema, ref.Batch(new.tolist(), kv.tolist(), 16, 4, 2, seed=B), f"{B} sequences")


def test_attention_low_bounds(ema):
    """max_len and max_q only size the call: true values past them give the same result."""
    b = ref.Batch([1, 50], [1500, 600], 32, 8, 2, seed=14)
    g = OnGpu(ema, b)
    import torch

    out = ema.paged_attention(g.q, g.cache, g.table, g.lengths, 8, q_starts=g.starts, max_q=1)
    torch.cuda.synchronize()
    ref.check_attention(down(out), *b.attention(), "low bounds")


def test_attention_lengths_past_the_table(ema):
    """Lengths are clamped to what the table holds, and negative ones to zero."""
    import torch

    b = ref.Batch([1, 1], [64, 32], 16, 4, 2, seed=15)
    g = OnGpu(ema, b)
    g.lengths.copy_(torch.tensor([5000, -7], dtype=torch.int32))
    out = down(g.attention())
    ref.check_attention(out[:1], *(x[:1] for x in b.attention()), "clamped")
    assert (out[1] == 0).all()


def test_rows_behind_the_last_sequence(ema):
    """Rows from q_starts[batch] on are neither read nor written, in a padded batch."""
    import torch

    b = ref.Batch([2, 1], [50, 20], 16, 8, 2, seed=16)
    g = OnGpu(ema, b)
    q = torch.cat([g.q, torch.full((6, 8, 128), float("nan"), dtype=torch.bfloat16, device="cuda")])
    out = torch.full((9, 8 * 128), 7.0, dtype=torch.bfloat16, device="cuda")
    ema.paged_attention(q, g.cache, g.table, g.lengths, 50, q_starts=g.starts, max_q=2, out=out)
    torch.cuda.synchronize()
    assert (out[3:] == 7.0).all()
    ref.check_attention(down(out[:3]), *b.attention(), "padded batch")


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("new,kv,prefix", [
    ([1] * 6, [50, 1, 33, 200, 64, 5], 0), ([40, 17, 90], [40, 200, 90], 0), ([260, 3], [300, 30], 0),
    ([1] * 6, [9] * 6, 70), ([1] * 40, [9] * 40, 300), ([2] * 130, [9] * 130, 130), ([1] * 40, [9] * 40, 3500),
    ([1] * 8, [0, 3] * 4, 17000),
])
def test_rows_that_are_not_finite(ema, new, kv, prefix, bad):
    """A query row that is not finite gives a row that is not finite, and no other row changes:
    neither its neighbours nor the other sequences'."""
    import torch

    b = ref.Batch(new, kv, 16, 8, 2, seed=31, prefix=prefix)
    g = OnGpu(ema, b)
    want = g.attention().clone()
    rows = [0, b.rows // 2, b.rows - 1]
    g.q[rows, 3, 17] = bad
    got = g.attention()
    torch.cuda.synchronize()
    hit = torch.zeros(b.rows, 8, dtype=torch.bool, device="cuda")
    hit[rows, 3] = True
    got, want = got.view(-1, 8, 128), want.view(-1, 8, 128)
    assert not torch.isfinite(got[hit]).all(-1).any()
    assert torch.isfinite(got[~hit]).all()
    ref.check_attention(down(got[~hit]), down(want[~hit]), down(want[~hit].abs()) + 1.0, "the other rows")


@pytest.mark.parametrize("new,kv,heads,prefix,pages", [
    ([1, 5, 30], [70, 300, 30], (8, 2), 0, "bf16"),              # segments
    ([1, 40], [70, 300], (8, 2), 0, "fp8"),
    ([700] * 6, [700, 701, 900, 760, 764, 3000], (8, 4), 0, "bf16"),  # blocks of 128 rows
    ([350, 480, 300, 129] * 18, [350, 500, 300, 400] * 18, (16, 2), 0, "bf16"),  # pairs of them
    ([1] * 6, [0, 5, 33, 1, 0, 90], (16, 8), 700, "bf16"),       # a prefix in every segment
    ([1] * 40, list(range(40)), (8, 2), 3300, "bf16"),           # once, in blocks
    ([1] * 6, [0, 5, 33, 1, 0, 90], (16, 8), 8000, "fp8"),       # once, in segments
])
def test_scores_far_below_zero(ema, new, kv, heads, prefix, pages):
    """Keys that share a large component against the queries: every score is near -97 (2^-140 before the
    row's max is taken off), and the softmax is what it is without the component."""
    import torch

    b = ref.Batch(new, kv, 16, *heads, seed=41, prefix=prefix)
    b.q[..., 0] = 10.0
    for x in [b.k, b.shared[0]] + [h[0] for h in b.held]:
        x[..., 0] = np.where(np.isnan(x[..., 0]), np.nan, -110.0)
    g = OnGpu(ema, b, pages)
    out = g.attention()
    torch.cuda.synchronize()
    # a score is at most 129 sums in 32 bits of up to 1100 in size, each off by 2^-14 at most; times
    # 128^-0.5 and for weight and row sum 2^-9.5 in all, 0.18 of the bound's 2^-7
    want, mag = b.attention()
    ref.check_attention(down(out), want, 1.18 * mag, f"scores far below zero {heads} {prefix} {pages}")


def test_prompt_sized_rows(ema):
    """Sequences of more rows than a segment, beside short ones, with and without row starts, and
    bounds below the truth (the sequences past them take another way)."""
    for new, kv in (([300, 1, 128, 0, 700], [300, 90, 1000, 0, 701]), ([129], [129]), ([400], [60]), ([2, 515], [2, 3000])):
        for heads in ((8, 2), (12, 1), (4, 4)):
            b = ref.Batch(new, kv, 16, *heads, seed=sum(new))
            run(ema, b, "prompts")
            run(ema, b, "prompts, not causal", causal=False)
            run(ema, b, "a low bound", max_q=200)
    for heads in ((16, 4), (5, 1)):
        run(ema, ref.Batch([250] * 5, [250, 400, 251, 1000, 333], 64, *heads, seed=3), "equal prompts", q_starts=None, max_q=None)


def test_prompts_of_many_sequences(ema):
    rng = np.random.default_rng(8)
    for B in (65, 200):
        new = rng.choice([0, 1, 2, 70, 150], B).tolist()
        kv = [n + int(rng.integers(0, 90)) for n in new]
        run(ema, ref.Batch(new, kv, 16, 4, 2, seed=B), f"{B} mixed sequences")
    # enough blocks for pairs of them
    new = rng.integers(300, 500, 70).tolist()
    run(ema, ref.Batch(new, new, 32, 16, 2, seed=5), "pairs of blocks")
    new[3], new[40], new[41] = 0, 1, 129
    run(ema, ref.Batch(new, [n + 60 for n in new], 16, 16, 2, seed=6), "pairs of blocks, ragged")
    run(ema, ref.Batch([600] * 24, [600] * 24, 16, 16, 2, seed=7), "equal pairs", q_starts=None, max_q=None)


def test_prompts_over_bad_pages_and_orders(ema):
    run(ema, ref.Batch([200, 3], [230, 50], 16, 8, 2, seed=9, holes=[(0, 0), (0, 7), (0, 14), (1, 1)]), "bad pages")
    for page in (32, 256):
        run(ema, ref.Batch([200, 310], [230, 400], page, 8, 2, seed=page), f"page {page}, nphd", order="nphd")


def test_uniform_rows(ema):
    """Without q_starts every sequence has n / B rows."""
    b = ref.Batch([4] * 3, [4, 90, 33], 16, 8, 2, seed=17)
    run(ema, b, "uniform rows", q_starts=None, max_q=None)


def test_workspace_across_shapes_and_repeats(ema):
    """One workspace for calls of different shapes, and the same call twice, bit for bit."""
    import torch

    ws = ema.paged_workspace(8, 512, 16, 2, 128, 64, 4096)
    first = None
    for new, kv in (([1] * 8, [4000] * 8), ([1], [3000]), ([40, 2], [40, 900]), ([1] * 8, [4000] * 8)):
        b = ref.Batch(new, kv, 32, 16, 2, seed=18)
        _, out = run(ema, b, "shared workspace", workspace=ws)
        if new == [1] * 8:
            assert first is None or torch.equal(first, out)
            first = out.clone()
    assert int(ws[:ema.EMA_DECODE_COUNTER_BYTES].max()) == 0  # the counters are zero again


def test_decode_workspace_is_shared(ema):
    """A paged call between two decode calls over the same workspace changes neither."""
    import torch

    ws = ema.paged_workspace(4, 4, 16, 2, 128, 1, 2048)
    ws = torch.zeros(max(ws.numel(), ema.decode_workspace_size(4, 16, 2, 128, 2048)), dtype=torch.uint8, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(3)
    k, v = (torch.randn(4, 2, 2048, 128, generator=gen, device="cuda").to(torch.bfloat16) for _ in range(2))
    cache = ema.StaticCache(4, 2, 2048, 128, k=k, v=v)
    q = torch.randn(4, 16, 128, generator=gen, device="cuda").to(torch.bfloat16)
    n = torch.tensor([2048, 1, 700, 64], dtype=torch.int32, device="cuda")
    want = ema.decode_attention(q, cache, n, 2048, workspace=ws).clone()
    run(ema, ref.Batch([1] * 4, [2000, 7, 900, 64], 64, 16, 2, seed=19), "between decode calls", workspace=ws)
    assert torch.equal(want, ema.decode_attention(q, cache, n, 2048, workspace=ws))


def test_static_cache_gives_the_same(ema):
    """The static cache's planes as pages: the same attention as ema_decode_attention, within the
    two kernels' roundings."""
    import torch

    B, Hkv, Hq, cap = 3, 2, 8, 512
    gen = torch.Generator(device="cuda").manual_seed(4)
    k, v = (torch.randn(B, Hkv, cap, 128, generator=gen, device="cuda").to(torch.bfloat16) for _ in range(2))
    q = torch.randn(B, Hq, 128, generator=gen, device="cuda").to(torch.bfloat16)
    n = torch.tensor([512, 17, 300], dtype=torch.int32, device="cuda")
    want = ema.decode_attention(q, ema.StaticCache(B, Hkv, cap, 128, k=k, v=v), n, cap)
    # pages of 64 positions of [B, Hkv, cap]: page i of sequence b at (b, :, 64 i)
    pk, pv = (x.view(B, Hkv, cap // 64, 64, 128).transpose(1, 2).reshape(-1, Hkv, 64, 128).contiguous() for x in (k, v))
    table = torch.arange(B * cap // 64, dtype=torch.int32, device="cuda").view(B, -1)
    got = ema.paged_attention(q, ema.PagedCache(pk.shape[0], Hkv, 64, 128, k=pk, v=pv), table, n, cap)
    d = (got.float() - want.float()).abs()
    # each within 2^-7 of weighted |v| (at most max |v| < 8) and one output rounding of the exact result
    assert d.max().item() <= 2 * (2 ** -7 * 8 + 2 ** -8 * want.float().abs().max().item())
    assert (d.norm() / want.float().norm()).item() < 2 ** -7


def test_streams_and_overlap(ema):
    """Two calls in flight on two streams, a workspace each; and a stream given by name."""
    import torch

    bs = [ref.Batch([1] * 6, [900] * 6, 16, 16, 2, seed=s) for s in (20, 21)]
    gs = [OnGpu(ema, b) for b in bs]
    ws = [ema.paged_workspace(6, 6, 16, 2, 128, 1, 900) for _ in bs]
    outs = [torch.empty(6, 16 * 128, dtype=torch.bfloat16, device="cuda") for _ in bs]
    streams = [torch.cuda.Stream() for _ in bs]
    torch.cuda.synchronize()
    for _ in range(5):
        for g, w, o, s in zip(gs, ws, outs, streams):
            g.attention(out=o, workspace=w, stream=s)
    torch.cuda.synchronize()
    for b, o in zip(bs, outs):
        ref.check_attention(down(o), *b.attention(), "two streams")


def test_stream_owns_what_the_call_allocates(ema):
    """A call on a stream of its own, the current stream busy and its free blocks full of ones: the
    call's workspace is cleared, and its output used, in the order of the call's stream."""
    import torch

    b = ref.Batch([1] * 3, [1800, 40, 900], 16, 16, 2, seed=22)
    g = OnGpu(ema, b)
    size = ema.paged_workspace_size(3, 3, 16, 2, 128, 1, 1800)
    s = torch.cuda.Stream()
    x = torch.ones(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    for _ in range(3):
        dirty = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        for _ in range(20):
            x.mul_(1.0)
        del dirty
        out = ema.paged_attention(g.q, g.cache, g.table, g.lengths, 1800, q_starts=g.starts, max_q=1, stream=s)
        s.synchronize()
        ref.check_attention(down(out), *b.attention(), "a stream's own workspace")
    torch.cuda.synchronize()


def test_captured_and_replayed(ema):
    """Append and attention in a graph, replayed over new inputs, lengths and tables, with eager
    work between; every replay against the eager result."""
    import torch

    Hq, Hkv, P, B = 16, 2, 32, 4
    gen = torch.Generator(device="cuda").manual_seed(5)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(torch.bfloat16)  # noqa: E731
    cache = ema.PagedCache(64, Hkv, P, 128, k=rnd(64, Hkv, P, 128), v=rnd(64, Hkv, P, 128))
    qkv, w = rnd(B, (Hq + 2 * Hkv) * 128), rnd(128)
    off = torch.zeros(B, dtype=torch.int32, device="cuda")
    n = torch.zeros(B, dtype=torch.int32, device="cuda")
    table = torch.zeros(B, 16, dtype=torch.int32, device="cuda")
    ws = [ema.paged_workspace(B, B, Hq, Hkv, 128, 1, 512) for _ in range(2)]
    q = torch.empty(B, Hq, 128, dtype=torch.bfloat16, device="cuda")
    out = torch.empty(B, Hq * 128, dtype=torch.bfloat16, device="cuda")

    def step(w_s, q, out):
        ema.paged_append(qkv, w, w, 1e-6, 1e6, off, Hq, cache, table, q_out=q)
        ema.paged_attention(q, cache, table, n, 512, out=out, workspace=w_s)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(ws[0], q, out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(ws[0], q, out)
    for i in range(4):
        qkv.copy_(rnd(*qkv.shape))
        off.copy_(torch.tensor([0, 31 + i, 200 * i % 500, 511 - i]))
        n.copy_(off + 1)
        table.copy_(torch.randperm(64, generator=gen, device="cuda")[:64].view(B, 16))
        g.replay()
        torch.cuda.synchronize()
        want_q, want = torch.empty_like(q), torch.empty_like(out)
        step(ws[1], want_q, want)
        torch.cuda.synchronize()
        assert torch.equal(q, want_q) and torch.equal(out, want), i


def test_pool_past_32_bits(ema):
    """Pages at offsets beyond 2^32 bytes and 2^31 elements."""
    import torch

    Hq, Hkv, P = 8, 8, 64
    n_pages = 40000  # 128 KiB each: 5 GB for K and for V
    b = ref.Batch([1, 3], [130, 70], P, Hq, Hkv, seed=22)
    g = OnGpu(ema, b)
    k, v = (torch.empty(n_pages, Hkv, P, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    used = sorted(set(b.table[b.table >= 0].tolist()))
    far = {p: n_pages - 1 - 700 * i for i, p in enumerate(used)}
    for p, f in far.items():
        k[f], v[f] = g.cache.k[p], g.cache.v[p]
    table = up(np.vectorize(lambda p: far.get(p, -1))(b.table).astype(np.int32))
    cache = ema.PagedCache(n_pages, Hkv, P, 128, k=k, v=v)
    out = ema.paged_attention(g.q, cache, table, g.lengths, 130, q_starts=g.starts, max_q=3)
    torch.cuda.synchronize()
    ref.check_attention(down(out), *b.attention(), "far pages")


# ------------------------------------------------------------------ shared prefix
@pytest.mark.parametrize("prefix", [1, 31, 64, 200, 1025])
@pytest.mark.parametrize("new,kv,heads", [
    ([1], [1], (8, 2)), ([1] * 4, [1, 40, 33, 0], (16, 8)), ([2, 1, 3, 0], [2, 90, 1, 0], (10, 2)),
    ([1] * 33, [5] * 33, (12, 1)), ([1] * 70, list(range(1, 71)), (8, 4)),
])
def test_prefix(ema, prefix, new, kv, heads):
    run(ema, ref.Batch(new, kv, 16, *heads, seed=prefix + len(new), prefix=prefix), f"prefix {prefix}")


@pytest.mark.parametrize("page", [16, 128])
def test_prefix_long(ema, page):
    run(ema, ref.Batch([1] * 9, [30] * 9, page, 40, 8, seed=1, prefix=4001), "long prefix")
    run(ema, ref.Batch([1] * 64, [3] * 64, page, 8, 2, seed=2, prefix=2500), "long prefix, 256 rows")


def test_prefix_ways(ema):
    """The three ways a prefix is read: its tiles in every segment (short ones), once in segments of
    few rows, once in blocks of 128 rows; each with sequences that hold nothing of their own."""
    for new, kv, heads, prefix in (([1] * 4, [0, 5, 33, 0], (8, 4), 200), ([1] * 6, [0, 5, 33, 1, 0, 90], (16, 8), 8000),
                                   ([2, 1, 0, 3], [2, 400, 7, 0], (10, 2), 40000), ([1] * 40, list(range(40)), (8, 2), 3300),
                                   ([3] * 30, [3] * 30, (12, 1), 10000)):
        run(ema, ref.Batch(new, kv, 64, *heads, seed=prefix, prefix=prefix), f"prefix {prefix}, {heads[0] // heads[1] * sum(new)} rows")
    run(ema, ref.Batch([1] * 6, [0, 5, 33, 1, 0, 90], 64, 16, 8, seed=1, prefix=8000), "prefix once, fp8", pages="fp8")


@pytest.mark.parametrize("held", [0, 1, 64, 129])
def test_prefix_shorter_than_its_bound(ema, held):
    """The prefix's length is on the device: what it holds counts, the bound only sizes the call."""
    import torch

    for n, heads in ((5, (16, 8)), (40, (8, 2))):
        b = ref.Batch([1] * n, [7] * n, 16, *heads, seed=held, prefix=held)
        g = OnGpu(ema, b)
        table = torch.full((600,), -1, dtype=torch.int32, device="cuda")
        if held:
            table[:g.prefix_table.numel()] = g.prefix_table
        out = ema.prefix_attention(g.q, g.cache, table, up(np.asarray([held], np.int32)), 9600, g.table, g.lengths, 7)
        torch.cuda.synchronize()
        ref.check_attention(down(out), *b.attention(), f"{held} of 9600")


def test_prefix_longer_than_its_bound(ema):
    """A prefix_len on the device past the call's bound counts as the bound, in every way of reading."""
    import torch

    for n, heads, bound, pages in ((4, (8, 4), 100, "bf16"), (6, (16, 8), 8000, "bf16"), (40, (8, 2), 3333, "bf16"),
                                   (6, (16, 8), 8000, "fp8")):
        b = ref.Batch([1] * n, [5] * n, 16, *heads, seed=bound, prefix=bound)
        g = OnGpu(ema, b, pages)
        g.prefix_len.fill_(bound + 3000)
        table = torch.cat([g.prefix_table, g.prefix_table]).contiguous()  # (pages for what it claims)
        out = ema.prefix_attention(g.q, g.cache, table, g.prefix_len, bound, g.table, g.lengths, 5)
        torch.cuda.synchronize()
        ref.check_attention(down(out), *b.attention(), f"bound {bound}")
        g.prefix_len.fill_(-5)
        out = ema.prefix_attention(g.q, g.cache, table, g.prefix_len, bound, g.table, g.lengths, 5)
        b.prefix, b.shared = 0, [x[:0] for x in b.shared]
        ref.check_attention(down(out), *b.attention(), "a negative length")


def test_wide_groups(ema):
    """More query heads per kv head than a segment or a block has rows."""
    for heads in ((40, 1), (144, 1), (256, 1)):
        run(ema, ref.Batch([1, 3, 2], [40, 3, 300], 16, *heads, seed=heads[0]), f"{heads[0]} heads on one")
    run(ema, ref.Batch([1, 1], [4, 9], 16, 144, 1, seed=2, prefix=90), "144 heads over a prefix")


def test_no_rows(ema):
    """Empty batches do nothing, whatever the addresses of empty tensors are."""
    import torch

    b = ref.Batch([1, 1], [5, 9], 16, 8, 2, seed=1)
    g = OnGpu(ema, b)
    zero = torch.zeros(3, dtype=torch.int32, device="cuda")
    q = torch.empty(0, 8, 128, dtype=torch.bfloat16, device="cuda")
    assert ema.paged_attention(q, g.cache, g.table, g.lengths, 9, q_starts=zero).shape == (0, 1024)
    qkv, w = torch.empty(0, 12 * 128, dtype=torch.bfloat16, device="cuda"), torch.ones(128, dtype=torch.bfloat16, device="cuda")
    before = g.cache.k.clone()
    assert ema.paged_append(qkv, w, w, 1e-6, 1e6, g.lengths, 8, g.cache, g.table, q_starts=zero).shape == (0, 8, 128)
    torch.cuda.synchronize()
    assert torch.equal(before.view(torch.int16), g.cache.k.view(torch.int16))
    # rows, but no sequence has any of them
    q = torch.randn(4, 8, 128, device="cuda").to(torch.bfloat16)
    out = torch.full((4, 1024), 7.0, dtype=torch.bfloat16, device="cuda")
    ema.paged_attention(q, g.cache, g.table, g.lengths, 9, q_starts=zero, max_q=1, out=out)
    torch.cuda.synchronize()
    assert (out == 7.0).all()


def test_prefix_fp8(ema):
    run(ema, ref.Batch([1] * 6, [1, 2, 3, 17, 33, 64], 16, 16, 4, seed=3, prefix=333), "fp8 prefix", pages="fp8")


def test_prefix_empty(ema):
    """A prefix that holds nothing (its length is on the device): the own pages alone."""
    import torch

    b = ref.Batch([1, 2, 1], [9, 80, 0], 16, 8, 2, seed=4)
    g = OnGpu(ema, b)
    out = ema.prefix_attention(g.q, g.cache, up(np.zeros(2, np.int32)), up(np.zeros(1, np.int32)), 32, g.table,
                               g.lengths, 80, q_starts=g.starts, max_q=2)
    torch.cuda.synchronize()
    ref.check_attention(down(out), *b.attention(), "empty prefix")


def test_prefix_rows_behind_the_last_sequence(ema):
    import torch

    b = ref.Batch([1, 2], [20, 5], 16, 8, 2, seed=5, prefix=100)
    g = OnGpu(ema, b)
    q = torch.cat([g.q, torch.full((40, 8, 128), float("nan"), dtype=torch.bfloat16, device="cuda")])
    out = torch.full((43, 8 * 128), 7.0, dtype=torch.bfloat16, device="cuda")
    ema.prefix_attention(q, g.cache, g.prefix_table, g.prefix_len, 100, g.table, g.lengths, 20, q_starts=g.starts,
                         max_q=2, out=out)
    torch.cuda.synchronize()
    assert (out[3:] == 7.0).all()
    ref.check_attention(down(out[:3]), *b.attention(), "padded batch over a prefix")


def test_prefix_equals_its_pages_in_every_table(ema):
    """The prefix as pages of every sequence's own table (whole pages): paged_attention over both
    gives the same, within the roundings of the two orders."""
    import torch

    b = ref.Batch([1] * 5, [7, 1, 64, 20, 33], 32, 16, 4, seed=6, prefix=256)
    g = OnGpu(ema, b)
    want, mag = b.attention()
    ref.check_attention(down(g.attention()), want, mag, "shared")
    table = torch.cat([g.prefix_table.expand(5, -1), g.table], 1).contiguous()
    out = ema.paged_attention(g.q, g.cache, table, g.lengths + 256, 320)
    ref.check_attention(down(out), want, mag, "in every table")


# ------------------------------------------------------------------ append
def append_case(ema, new, off, page, Hq, Hkv, D=128, seed=0, pages="bf16", flags=0, prefix=0, order="nhpd", bad=(),
                starts=True, theta=1e6, pad=0):
    """One append against float64; every slot that no row is written to keeps its bits."""
    import torch

    rng = np.random.default_rng(seed)
    kv = [n + o for n, o in zip(new, off)]
    b = ref.Batch(new, kv, page, Hq, Hkv, seed, D=D)
    for i, (s, p) in enumerate(bad):
        b.table[s, p] = (-1, b.n_pages, 1 << 30)[i % 3]
    H = Hq + 2 * Hkv
    qkv = ref.normal(rng, b.rows + pad, H, D)
    qw, kw = (ref.bf16(1 + 0.1 * rng.standard_normal(D)) for _ in range(2))
    b.k, b.v = ref.normal(rng, *b.k.shape), ref.normal(rng, *b.v.shape)
    g = OnGpu(ema, b, pages, order)
    before = [x.clone() for x in (g.cache.k, g.cache.v)]
    q_out = torch.full((b.rows + pad, Hq, D), 7.0, dtype=torch.bfloat16, device="cuda")
    say(f"append new {new[:6]} off {off[:6]} page {page} {Hq}q/{Hkv}kv D {D} {pages}")
    ema.paged_append(up(qkv.reshape(b.rows + pad, -1)), up(qw), up(kw), 1e-6, theta,
                     up(np.asarray(off, np.int32)), Hq, g.cache, g.table, q_starts=g.starts if starts else None,
                     flags=flags, q_out=q_out, prefix_len=up(np.asarray([prefix], np.int32)) if prefix else None)
    torch.cuda.synchronize()
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    if not flags & (ema.EMA_PRE_NO_NORM | ema.EMA_PRE_NO_Q_NORM):
        q = ref.norm(q, qw, 1e-6)
    if not flags & (ema.EMA_PRE_NO_NORM | ema.EMA_PRE_NO_K_NORM):
        k = ref.norm(k, kw, 1e-6)
    pos = np.concatenate([o + np.arange(n) for n, o in zip(new, off)] + [np.zeros(pad)]).astype(np.int64)
    if not flags & ema.EMA_PRE_NO_ROPE:
        q, k = ref.rotate(q, pos + prefix, theta), ref.rotate(k, pos + prefix, theta)

    def close(got, want, what, extra=0.0):
        # one rounding to bf16 (2^-8), and 32-bit arithmetic on values of a few units (2^-20)
        bound = 2.0 ** -8 * np.abs(want) + 2.0 ** -20 * max(1.0, np.abs(want).max(initial=0)) + extra
        d = np.abs(got - want)
        assert (d <= bound).all(), f"{what}: {(d / bound).max()} of the bound"

    n = b.rows
    close(down(q_out)[:n], q[:n], "q")
    assert (q_out[n:] == 7.0).all()
    got = [x.cpu() for x in (g.cache.k, g.cache.v)]
    written = np.zeros(b.k.shape[:1] + b.k.shape[2:3], bool)  # (page, slot)
    seq = np.repeat(np.arange(len(new)), new)
    pages_np = b.table[seq, np.minimum(np.maximum(pos[:n], 0) // page, b.table.shape[1] - 1)]
    ok = (pos[:n] >= 0) & (pos[:n] // page < b.table.shape[1]) & (pages_np >= 0) & (pages_np < b.n_pages)
    pg, sl = pages_np[ok], pos[:n][ok] % page
    written[pg, sl] = True
    for name, x, want, was in (("k", got[0], k, before[0]), ("v", got[1], v, before[1])):
        xs = x.transpose(1, 2)[pg, sl]  # [rows, Hkv, D]
        if pages == "fp8":
            e = (g.cache.k_exp if name == "k" else g.cache.v_exp).cpu().transpose(1, 2)[pg, sl].numpy().astype(np.float64)
            val = xs.view(torch.float8_e4m3fn).double().numpy().reshape(-1, Hkv, D // 64, 64) * 2.0 ** e[..., None]
            w = want[:n][ok].reshape(-1, Hkv, D // 64, 64)
            # half a step of e4m3: 2^-4 of a normal value, 2^-10 of the scale below; the bf16 row first
            bound = (2.0 ** -4 + 2.0 ** -8) * np.abs(w) + 2.0 ** -10 * 2.0 ** e[..., None] + 2.0 ** -20
            assert (np.abs(val - w) <= bound).all(), name
            top = np.abs(w).max(-1)
            assert (e >= np.ceil(np.log2(top * (1 - 2.0 ** -8) / 448))).all() and (e <= np.ceil(np.log2(top * (1 + 2.0 ** -8) / 448))).all()
        elif name == "v":
            assert (xs.double().numpy() == v[:n][ok]).all()
        else:
            close(xs.double().numpy(), want[:n][ok], name)
        same = (x == was.cpu()).transpose(1, 2).all(-1).all(-1).numpy()
        assert same[~written].all(), f"{name}: a slot outside the call changed"
    return g


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("heads", [(16, 8), (4, 4), (12, 1), (40, 8)])
def test_append(ema, D, heads):
    append_case(ema, [1], [0], 16, *heads, D=D)
    append_case(ema, [1, 1, 1], [5, 15, 16], 16, *heads, D=D, starts=False)
    append_case(ema, [17, 0, 1, 40], [0, 3, 63, 7], 32, *heads, D=D)


@pytest.mark.parametrize("flags", [0, 1, 2, 3, 8, 16, 8 | 2])
def test_append_flags(ema, flags):
    append_case(ema, [3, 1], [30, 0], 16, 8, 2, flags=flags)


@pytest.mark.parametrize("page", [16, 128, 1024])
def test_append_orders(ema, page):
    append_case(ema, [20, 3], [5, 100], page, 8, 2, order="nphd")


@pytest.mark.parametrize("page", [16, 64])
def test_append_fp8(ema, page):
    append_case(ema, [20, 1, 2], [5, 100, 0], page, 8, 2, pages="fp8")


@pytest.mark.parametrize("theta", [1e4, 1e6, 5e5])
def test_append_far_positions(ema, theta):
    """Angles of far positions keep their accuracy (a prefix stands before the own positions)."""
    append_case(ema, [4, 2], [12, 0], 16, 8, 2, prefix=131071, theta=theta)
    append_case(ema, [4, 2], [12, 0], 16, 8, 2, prefix=(1 << 30) + 12345, theta=theta)


def test_append_bad_pages_and_padding(ema):
    append_case(ema, [40, 20], [0, 12], 16, 8, 2, bad=[(0, 1), (1, 0), (1, 1)])
    append_case(ema, [4, 2], [3, 12], 16, 8, 2, pad=5)


def test_append_outside_the_table(ema):
    """Rows at negative positions, or past the table, get their q and are not stored."""
    import torch

    b = ref.Batch([1] * 3, [16, 16, 16], 16, 8, 2, 0)
    b.k, b.v = (ref.normal(np.random.default_rng(1), *b.k.shape) for _ in range(2))
    g = OnGpu(ema, b)
    before = g.cache.k.clone(), g.cache.v.clone()
    qkv = torch.randn(3, 12 * 128, device="cuda").to(torch.bfloat16)
    w = torch.ones(128, dtype=torch.bfloat16, device="cuda")
    off = up(np.asarray([-1, 16, 2147483647], np.int32))
    q = ema.paged_append(qkv, w, w, 1e-6, 1e6, off, 8, g.cache, g.table)
    torch.cuda.synchronize()
    assert torch.equal(g.cache.k, before[0]) and torch.equal(g.cache.v, before[1])
    x = ref.norm(down(qkv).reshape(3, 12, 128)[:, :8], np.ones(128), 1e-6)
    want = ref.rotate(x, np.asarray([-1, 16, 2147483647]), 1e6)
    assert (np.abs(down(q) - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -18).all()


@pytest.mark.parametrize("B", [64, 65, 300, 1024])
def test_append_many_sequences(ema, B):
    rng = np.random.default_rng(B)
    append_case(ema, rng.integers(0, 4, B).tolist(), rng.integers(0, 40, B).tolist(), 16, 4, 2, seed=B)


# ------------------------------------------------------------------ as they are used
@pytest.mark.parametrize("pages", ["bf16", "fp8"])
def test_prompt_then_tokens(ema, pages):
    """Ragged prompts, then drafted and single tokens, appended and attended call by call over one
    pool, against float64 attention over what the pool holds; then more samples of the first
    sequence's prompt as a shared prefix."""
    import torch

    Hq, Hkv, D, P, B = 8, 2, 128, 16, 3
    rng = np.random.default_rng(9)
    cols, n_pages = 12, 50
    cache = ema.PagedCache(n_pages, Hkv, P, D, dtype=pages)
    table = torch.from_numpy(rng.permutation(n_pages)[:B * cols].reshape(B, cols).astype(np.int32)).cuda()
    w = [up(ref.bf16(1 + 0.1 * rng.standard_normal(D))) for _ in range(2)]
    ws = ema.paged_workspace(8, 256, Hq, Hkv, D, 128, cols * P, max_prefix=cols * P)

    def held(pages_of, n):
        """Positions [0, n) as the pool holds them, [n, Hkv, D] twice."""
        out = []
        for x, e in ((cache.k, cache.k_exp), (cache.v, cache.v_exp)):
            y = x[pages_of.long()].cpu()
            if pages == "fp8":
                y = y.view(torch.float8_e4m3fn).double().unflatten(-1, (-1, 64)) * torch.exp2(e[pages_of.long()].cpu().double())[..., None]
                y = y.flatten(-2)
            out.append(y.double().transpose(1, 2).reshape(-1, Hkv, D)[:n].numpy())
        return out

    kv = [0] * B
    for new in ([37, 80, 1], [1, 1, 1], [4, 1, 3], [1, 1, 1]):
        n = sum(new)
        starts = up(np.concatenate([[0], np.cumsum(new)]).astype(np.int32))
        off = up(np.asarray(kv, np.int32))
        qkv = up(ref.normal(rng, n, (Hq + 2 * Hkv) * D))
        q = ema.paged_append(qkv, *w, 1e-6, 1e6, off, Hq, cache, table, q_starts=starts)
        kv = [a + b for a, b in zip(kv, new)]
        out = ema.paged_attention(q, cache, table, up(np.asarray(kv, np.int32)), max(kv), q_starts=starts, max_q=max(new),
                                  workspace=ws)
        torch.cuda.synchronize()
        at = 0
        for b in range(B):
            o, m = ref.attend(down(q)[at:at + new[b]], *held(table[b], kv[b]), kv[b] - new[b] + np.arange(new[b]), D ** -0.5)
            ref.check_attention(down(out)[at:at + new[b]], o.reshape(new[b], -1), m.reshape(new[b], -1), f"sequence {b} at {kv[b]}")
            at += new[b]
    # four samples that continue sequence 0
    S = 4
    free = [p for p in range(n_pages) if p not in set(table.cpu().numpy().ravel().tolist())]
    own = torch.tensor(free[:S * 2], dtype=torch.int32, device="cuda").view(S, 2)
    plen = up(np.asarray([kv[0]], np.int32))
    for t in range(3):
        off = up(np.full(S, t, np.int32))
        q = ema.paged_append(up(ref.normal(rng, S, (Hq + 2 * Hkv) * D)), *w, 1e-6, 1e6, off, Hq, cache, own, prefix_len=plen)
        out = ema.prefix_attention(q, cache, table[0].contiguous(), plen, kv[0], own, off + 1, t + 1, workspace=ws)
        torch.cuda.synchronize()
        shared = held(table[0], kv[0])
        for s in range(S):
            k, v = (np.concatenate([a, b]) for a, b in zip(shared, held(own[s], t + 1)))
            o, m = ref.attend(down(q)[s:s + 1], k, v, [kv[0] + t], D ** -0.5)
            ref.check_attention(down(out)[s:s + 1], o.reshape(1, -1), m.reshape(1, -1), f"sample {s} token {t}")
