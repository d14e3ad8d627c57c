"""Paged cache on the GPU: what its header allows beyond the ordinary calls of test_gpu_paged.py.
Bad entries in a shared prefix, FP8 pages in other orders, prompts behind a prefix, padded batches,
captured calls of every way of reading; against plain float64 (tests/paged_ref.py)."""
import numpy as np
import pytest

import paged_ref as ref
from gpu_util import say
from test_gpu_paged import OnGpu, down, ema, run, up  # noqa: F401 (ema: the fixture)

pytestmark = pytest.mark.gpu

# new rows, positions held, heads, prefix, pages: each way in which keys are read
WAYS = {
    "segments": ([1, 5, 0, 30], [70, 300, 12, 30], (8, 2), 0, "bf16"),
    "segments fp8": ([1, 5, 0, 30], [70, 300, 12, 30], (8, 2), 0, "fp8"),
    "blocks": ([500, 1, 700, 650, 333], [500, 90, 900, 650, 400], (8, 8), 0, "bf16"),
    "pairs": ([350, 480, 300, 129] * 18, [350, 500, 300, 400] * 18, (16, 2), 0, "bf16"),
    "prefix in segments": ([1] * 4, [0, 5, 33, 0], (8, 4), 200, "bf16"),
    "prefix in segments fp8": ([1] * 4, [0, 5, 33, 0], (8, 4), 200, "fp8"),
    "prefix in blocks": ([1] * 40, list(range(40)), (8, 2), 3300, "bf16"),
    "prefix once fp8": ([1] * 6, [0, 5, 33, 1, 0, 90], (16, 8), 8000, "fp8"),
}


def with_prefix(*names):
    return [n for n in WAYS if WAYS[n][3] and (not names or n in names)]


def batch(name, seed, page=16):
    new, kv, heads, prefix, pages = WAYS[name]
    return ref.Batch(new, kv, page, *heads, seed=seed, prefix=prefix), pages


@pytest.mark.parametrize("way", with_prefix())
def test_bad_pages_in_a_prefix(ema, way):
    """Entries of the prefix's table outside the pool, first, middle and last: zero rows."""
    b, pages = batch(way, 51)
    last = -(-b.prefix // b.page) - 1
    for p, bad in ((0, -1), (last // 2, b.n_pages), (last // 2 + 1, 1 << 30), (last, -(1 << 31))):
        b.prefix_table[p] = bad
        for x in b.shared:
            x[p * b.page:(p + 1) * b.page] = 0.0
    run(ema, b, way, pages=pages)


@pytest.mark.parametrize("way", ["segments fp8", "prefix in segments fp8", "prefix once fp8"])
@pytest.mark.parametrize("page", [16, 64])
def test_fp8_pages_in_another_order(ema, way, page):
    """FP8 codes as [page, position, head, D] in memory: the same bits as [page, head, position, D]."""
    import torch

    b, pages = batch(way, 52, page)
    g, want = run(ema, b, way, pages=pages)
    c = g.cache
    k, v = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (c.k, c.v))
    g.cache = ema.PagedCache(b.n_pages, b.Hkv, b.page, b.D, k=k, v=v, dtype="fp8", k_exp=c.k_exp, v_exp=c.v_exp)
    assert g.cache.desc.stride_head == 128 and g.cache.desc.stride_pos == 128 * b.Hkv
    assert torch.equal(want, g.attention())


def test_append_to_fp8_pages_in_another_order(ema):
    import torch

    gen = torch.Generator(device="cuda").manual_seed(53)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(torch.bfloat16)  # noqa: E731
    Hq, Hkv, P, n_pages = 8, 4, 32, 12
    qkv, w = rnd(40, (Hq + 2 * Hkv) * 128), rnd(128)
    starts, off = up(np.array([0, 33, 33, 40], np.int32)), up(np.array([30, 4, 90], np.int32))
    table = up(np.array([[3, 1, 7, -1], [5, -1, -1, -1], [0, 2, 9, 11]], np.int32))
    new = lambda *s: torch.full(s, 0x33, dtype=torch.uint8, device="cuda")  # noqa: E731
    pools = []
    for order in ("nhpd", "nphd"):
        kv = [new(n_pages, Hkv, P, 128) if order == "nhpd" else new(n_pages, P, Hkv, 128).transpose(1, 2) for _ in range(2)]
        ex = [torch.full((n_pages, Hkv, P, 2), 5, dtype=torch.int8, device="cuda") for _ in range(2)]
        c = ema.PagedCache(n_pages, Hkv, P, 128, k=kv[0], v=kv[1], dtype="fp8", k_exp=ex[0], v_exp=ex[1])
        q = ema.paged_append(qkv, w, w, 1e-6, 1e6, off, Hq, c, table, q_starts=starts)
        pools.append((q, *kv, *ex))
    torch.cuda.synchronize()
    for a, b in zip(*pools):  # (pools that test_gpu_paged.py holds against float64 in the first order)
        assert torch.equal(a, b)
    assert (pools[0][1] != 0x33).any()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("way", [w for w in WAYS if w != "pairs"])
def test_other_rows_keep_their_attention(ema, way, bad):
    """Query rows that are not finite: every other row within the ordinary bound of its own values."""
    import torch

    b, pages = batch(way, 54)
    g = OnGpu(ema, b, pages)
    say(f"rows of {bad}, {way}")
    rows = [0, b.rows // 2, b.rows - 1]
    g.q[rows, 3, 17] = bad
    got = g.attention().view(-1, b.Hq, 128)
    torch.cuda.synchronize()
    want, mag = (x.reshape(-1, b.Hq, 128) for x in b.attention())
    hit = np.zeros((b.rows, b.Hq), bool)
    hit[rows, 3] = True
    seq = np.repeat(np.arange(len(b.new)), b.new)  # (a row that sees no key is zeros whatever it holds)
    keys = b.prefix + np.asarray(b.kv)[seq] > 0
    assert not np.isfinite(down(got))[hit & keys[:, None]].all(-1).any()
    ref.check_attention(down(got)[~hit], want[~hit], mag[~hit], "the other rows")


@pytest.mark.parametrize("pages", ["bf16", "fp8"])
@pytest.mark.parametrize("prefix", [100, 3301])
@pytest.mark.parametrize("heads", [(8, 2), (12, 1), (4, 4)])
def test_prompts_behind_a_prefix(ema, heads, prefix, pages):
    run(ema, ref.Batch([200, 1, 70, 0], [200, 40, 333, 5], 32, *heads, seed=55, prefix=prefix), "prompts behind a prefix",
        pages=pages)
    run(ema, ref.Batch([150] * 3, [150, 3, 400], 16, *heads, seed=56, prefix=prefix), "equal prompts behind a prefix",
        pages=pages, q_starts=None, max_q=None)  # (3 positions for 150 rows: most see the prefix alone)


@pytest.mark.parametrize("way", list(WAYS))
def test_rows_before_the_first_and_behind_the_last_sequence(ema, way):
    """Row starts that begin past 0 and end before the packed rows do: the rows outside are NaN and
    stay out of every sequence; their output is not written."""
    import torch

    b, pages = batch(way, 57)
    g = OnGpu(ema, b, pages)
    say(f"padded on both sides, {way}")
    pad = lambda n: torch.full((n, b.Hq, 128), float("nan"), dtype=torch.bfloat16, device="cuda")  # noqa: E731
    g.q = torch.cat([pad(3), g.q, pad(140)])
    g.starts = g.starts + 3
    out = torch.full((b.rows + 143, b.Hq * 128), 7.0, dtype=torch.bfloat16, device="cuda")
    g.attention(out=out)
    torch.cuda.synchronize()
    assert (out[:3] == 7.0).all() and (out[b.rows + 3:] == 7.0).all()
    ref.check_attention(down(out[3:b.rows + 3]), *b.attention(), way)


@pytest.mark.parametrize("scale", [0.01, 1.0])
@pytest.mark.parametrize("way", ["blocks", "prefix in segments", "prefix in blocks", "prefix once fp8"])
def test_scales(ema, way, scale):
    b, pages = batch(way, 58)
    run(ema, b, f"{way}, scale {scale}", pages=pages, scale=scale)


@pytest.mark.parametrize("way", ["segments", "blocks", "prefix in segments", "prefix in blocks"])
def test_pool_past_32_bits_every_way(ema, way):
    """Pages at offsets beyond 2^32 bytes and 2^31 elements, of the sequences and of the prefix."""
    import torch

    b, _ = batch(way, 59, page=64)
    g = OnGpu(ema, b)
    n_pages = (6 << 30) // (b.Hkv * 64 * 128 * 2)  # 6 GiB for K and for V
    k, v = (torch.empty(n_pages, b.Hkv, 64, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    far = lambda p: n_pages - 1 - p * ((n_pages - 1) // b.n_pages)  # noqa: E731
    at = torch.arange(b.n_pages, device="cuda")
    k[far(at)], v[far(at)] = g.cache.k, g.cache.v
    g.cache = ema.PagedCache(n_pages, b.Hkv, 64, 128, k=k, v=v)
    g.table = torch.where(g.table >= 0, far(g.table), g.table).to(torch.int32)
    if b.prefix:
        g.prefix_table = far(g.prefix_table).to(torch.int32)
    out = g.attention()
    torch.cuda.synchronize()
    ref.check_attention(down(out), *b.attention(), way)


@pytest.mark.parametrize("way", list(WAYS))
def test_captured_every_way(ema, way):
    """Captured with a workspace of its own and with one that the call makes itself; replayed over new
    queries and lengths with eager work between, every replay against the eager result, bit for bit."""
    import torch

    b, pages = batch(way, 60)
    g = OnGpu(ema, b, pages)
    say(f"captured, {way}")
    outs = [torch.empty(b.rows, b.Hq * 128, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    size = ema.paged_workspace_size(len(b.new), b.rows, b.Hq, b.Hkv, 128, max(b.new), max(b.kv), b.prefix)
    ws = torch.zeros(size, dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        g.attention(out=outs[0], workspace=ws)
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for graph, out, w in zip(graphs, outs, (ws, None)):
        with torch.cuda.graph(graph):
            g.attention(out=out, workspace=w)
    lengths = g.lengths.clone()
    for i in range(4):
        g.q.copy_(torch.randn(g.q.shape, device="cuda"))
        g.lengths.copy_((lengths - i).clamp(min=0))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = g.attention()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want), i


@pytest.mark.parametrize("way", with_prefix())
def test_nothing_of_their_own(ema, way):
    """Every sequence at length 0, table rows of no page: the prefix alone."""
    new, _, heads, prefix, pages = WAYS[way]
    run(ema, ref.Batch(new, [0] * len(new), 16, *heads, seed=61, prefix=prefix), way, pages=pages)
