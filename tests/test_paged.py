"""Paged cache without a GPU: the kernels' integer parts (tests/cpp/test_paged.cpp) and the calls
that are refused on the host, before any HIP call, with the documented codes."""
import ctypes
import os
import random
import re
import subprocess

import pytest

CPP = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp")
P = 0x40000  # an aligned address that no refused call touches


def test_integer_parts():
    subprocess.run(["make", "-s", "-C", CPP, "test_paged"], check=True)
    r = subprocess.run([os.path.join(CPP, "test_paged")], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "checks passed" in r.stdout, r.stdout + r.stderr


@pytest.fixture(scope="module")
def ema():
    import ema_attn

    ema_attn.lib()
    return ema_attn


def pool(ema, n_pages=10, Hkv=8, page=16, D=128, **over):
    d = ema.KvCacheDesc()
    if over.pop("fp8", False):
        rc = ema.lib().ema_kvcache_init_fp8(ctypes.byref(d), P, P, P, P, n_pages, Hkv, page, D, over.pop("n_rot", 0))
    else:
        rc = ema.lib().ema_kvcache_init(ctypes.byref(d), P, P, n_pages, Hkv, page, D)
    assert rc == ema.EMA_OK, ema.last_error()
    for k, v in over.items():
        setattr(d, k, v)
    return d


def append(ema, d, **over):
    a = dict(qkv=P, qw=P, kw=P, eps=1e-6, theta=1e6, starts=P, off=P, prefix=None, batch=2, rows=5, heads=16, flags=0,
             q=P, table=P, cols=4)
    assert not set(over) - set(a)
    a.update(over)
    return ema.lib().ema_paged_append(None, a["qkv"], a["qw"], a["kw"], a["eps"], a["theta"], a["starts"], a["off"],
                                      a["prefix"], a["batch"], a["rows"], a["heads"], a["flags"], a["q"],
                                      ctypes.byref(d) if d is not None else None, a["table"], a["cols"])


def attend(ema, d, prefix=False, **over):
    a = dict(q=P, table=P, cols=4, starts=P, lengths=P, batch=2, rows=5, max_q=3, max_len=64, heads=16, scale=0.1,
             flags=1, out=P, ws=P, bytes=1 << 40, ptable=P, pcols=3, plen=P, max_prefix=48)
    assert not set(over) - set(a)
    a.update(over)
    ref = ctypes.byref(d) if d is not None else None
    if prefix:
        return ema.lib().ema_prefix_attention(None, a["q"], ref, a["ptable"], a["pcols"], a["plen"], a["max_prefix"],
                                              a["table"], a["cols"], a["starts"], a["lengths"], a["batch"], a["rows"],
                                              a["max_q"], a["max_len"], a["heads"], a["scale"], a["out"], a["ws"], a["bytes"])
    return ema.lib().ema_paged_attention(None, a["q"], ref, a["table"], a["cols"], a["starts"], a["lengths"], a["batch"],
                                         a["rows"], a["max_q"], a["max_len"], a["heads"], a["scale"], a["flags"], a["out"],
                                         a["ws"], a["bytes"])


def test_pools_that_are_refused(ema):
    calls = (append, attend, lambda e, d: attend(e, d, prefix=True))
    for call in calls:
        assert call(ema, None) == ema.EMA_ERR_INVALID_ARG
        for page in (8, 24, 48, 100):
            assert call(ema, pool(ema, page=page)) == ema.EMA_ERR_UNSUPPORTED and "power of two" in ema.last_error()
        assert call(ema, pool(ema, fp8=True, n_rot=64)) == ema.EMA_ERR_UNSUPPORTED
        assert call(ema, pool(ema, flags=ema.EMA_KV_ROTATING)) == ema.EMA_ERR_INVALID_ARG
        assert call(ema, pool(ema, k=None)) == ema.EMA_ERR_INVALID_ARG
        assert call(ema, pool(ema, k=P + 8)) == ema.EMA_ERR_INVALID_ARG
        assert call(ema, pool(ema, fp8=True, k_exp=P + 1)) == ema.EMA_ERR_INVALID_ARG
        assert call(ema, pool(ema, stride_pos=64)) == ema.EMA_ERR_SHAPE
        assert call(ema, pool(ema, stride_pos=1 << 26)) == ema.EMA_ERR_UNSUPPORTED
        assert call(ema, pool(ema, stride_batch=1 << 31)) == ema.EMA_ERR_UNSUPPORTED
        assert call(ema, pool(ema, stride_head=1 << 31)) == ema.EMA_ERR_UNSUPPORTED
        d = ema.KvCacheDesc()
        assert ema.lib().ema_kvcache_init_int4(ctypes.byref(d), P, P, P, P, P, P, 10, 8, 32, 128) == ema.EMA_OK
        assert call(ema, d) == ema.EMA_ERR_UNSUPPORTED


def test_appends_that_are_refused(ema):
    d = pool(ema)
    for name in ("qkv", "off", "q", "table", "qw", "kw"):
        assert append(ema, d, **{name: None}) == ema.EMA_ERR_INVALID_ARG, name
    for name in ("qkv", "q", "qw", "kw"):
        assert append(ema, d, **{name: P + 8}) == ema.EMA_ERR_INVALID_ARG, name
    assert append(ema, d, flags=4) == ema.EMA_ERR_INVALID_ARG
    assert append(ema, d, heads=12) == ema.EMA_ERR_SHAPE
    assert append(ema, d, heads=0) == ema.EMA_ERR_SHAPE
    assert append(ema, d, cols=0) == ema.EMA_ERR_SHAPE
    assert append(ema, d, batch=0) == ema.EMA_ERR_SHAPE
    assert append(ema, d, rows=-1) == ema.EMA_ERR_SHAPE
    assert append(ema, d, starts=None) == ema.EMA_ERR_SHAPE and "q_starts" in ema.last_error()  # 5 rows of 2 sequences
    assert append(ema, d, batch=1025) == ema.EMA_ERR_UNSUPPORTED
    assert append(ema, d, rows=1 << 20) == ema.EMA_ERR_SHAPE
    assert append(ema, d, cols=(1 << 26) + 1) == ema.EMA_ERR_UNSUPPORTED
    assert append(ema, d, theta=float("inf")) == ema.EMA_ERR_INVALID_ARG
    assert append(ema, d, eps=-1.0) == ema.EMA_ERR_INVALID_ARG
    assert append(ema, d, theta=0.0) == ema.EMA_ERR_INVALID_ARG
    assert append(ema, d, theta=float("nan")) == ema.EMA_ERR_INVALID_ARG
    assert append(ema, pool(ema, D=96)) == ema.EMA_ERR_UNSUPPORTED
    # nothing to do: no launch
    assert append(ema, d, rows=0) == ema.EMA_OK
    assert append(ema, d, rows=0, qkv=None, q=None) == ema.EMA_OK  # what an empty tensor's address is
    assert append(ema, d, rows=0, qw=None, flags=ema.EMA_PRE_NO_Q_NORM) == ema.EMA_OK


@pytest.mark.parametrize("prefix", [False, True])
def test_attention_that_is_refused(ema, prefix):
    d = pool(ema)
    for name in ("q", "out", "lengths", "table"):
        assert attend(ema, d, prefix, **{name: None}) == ema.EMA_ERR_INVALID_ARG, name
    for name in ("q", "out", "ws"):
        assert attend(ema, d, prefix, **{name: P + 4}) == ema.EMA_ERR_INVALID_ARG, name
    assert attend(ema, d, prefix, heads=12) == ema.EMA_ERR_SHAPE
    assert attend(ema, pool(ema, Hkv=1), prefix, heads=257) == ema.EMA_ERR_UNSUPPORTED
    assert attend(ema, d, prefix, cols=0) == ema.EMA_ERR_SHAPE
    assert attend(ema, d, prefix, starts=None) == ema.EMA_ERR_SHAPE
    assert attend(ema, d, prefix, batch=1025) == ema.EMA_ERR_UNSUPPORTED
    assert attend(ema, d, prefix, max_q=-1) == ema.EMA_ERR_SHAPE
    assert attend(ema, d, prefix, max_len=65) == ema.EMA_ERR_CAPACITY  # 4 pages of 16
    assert attend(ema, d, prefix, max_len=-1) == ema.EMA_ERR_CAPACITY
    for scale in (0.0, -1.0, float("nan")):
        assert attend(ema, d, prefix, scale=scale) == ema.EMA_ERR_INVALID_ARG
    assert attend(ema, d, prefix, ws=None) == ema.EMA_ERR_WORKSPACE
    assert attend(ema, d, prefix, bytes=1000) == ema.EMA_ERR_WORKSPACE
    assert attend(ema, pool(ema, D=64), prefix) == ema.EMA_ERR_UNSUPPORTED
    # more key tiles over all row blocks than the kernels count
    assert attend(ema, pool(ema, page=4096), prefix, cols=1 << 18, rows=1 << 18) == ema.EMA_ERR_UNSUPPORTED
    assert attend(ema, d, prefix, rows=0) == ema.EMA_OK
    assert attend(ema, d, prefix, rows=0, q=None, out=None) == ema.EMA_OK
    if prefix:
        assert attend(ema, d, True, ptable=None) == ema.EMA_ERR_INVALID_ARG
        assert attend(ema, d, True, plen=None) == ema.EMA_ERR_INVALID_ARG
        assert attend(ema, d, True, pcols=0) == ema.EMA_ERR_SHAPE
        assert attend(ema, d, True, max_prefix=49) == ema.EMA_ERR_CAPACITY
        assert attend(ema, d, True, max_prefix=0) == ema.EMA_ERR_CAPACITY
    else:
        assert attend(ema, d, flags=2) == ema.EMA_ERR_INVALID_ARG


def test_workspace_sizes(ema):
    n = ema.paged_workspace_size(32, 32, 32, 8, 128, 1, 8192)
    assert n > ema.EMA_DECODE_COUNTER_BYTES
    assert ema.paged_workspace_size(32, 32, 32, 8, 128, 1, 8192, 4096) > n
    for bad, code in ((dict(head_dim=64), ema.EMA_ERR_UNSUPPORTED), (dict(batch=0), ema.EMA_ERR_SHAPE),
                      (dict(n_heads=9), ema.EMA_ERR_SHAPE), (dict(max_len=-1), ema.EMA_ERR_SHAPE),
                      (dict(max_prefix=-1), ema.EMA_ERR_SHAPE), (dict(max_q=-1), ema.EMA_ERR_SHAPE)):
        a = dict(batch=2, n_rows=2, n_heads=16, n_kv_heads=8, head_dim=128, max_q=1, max_len=64, max_prefix=0)
        a.update(bad)
        with pytest.raises(ema.EmaError) as e:
            ema.paged_workspace_size(**a)
        assert e.value.code == code, bad


def test_pages_whose_positions_span_too_much(ema):
    """Positions outermost in the pool: the offset of a position within its page is 32 bits of bytes
    in the prompts' kernel."""
    for fp8 in (False, True):
        for call in (append, attend, lambda e, d, **o: attend(e, d, prefix=True, **o)):
            over = dict(fp8=fp8, page=1024, stride_batch=128, stride_head=1280)
            d = pool(ema, stride_pos=1 << 22, **over)
            assert call(ema, d, rows=0) == ema.EMA_ERR_UNSUPPORTED and "span" in ema.last_error()
            assert call(ema, pool(ema, stride_pos=1 << 21, **over), rows=0) == ema.EMA_OK


def needed(ema, **over):
    """Bytes that a call asks for, from its refusal without a workspace."""
    assert attend(ema, pool(ema, Hkv=over.pop("hkv"), page=4096), over.pop("prefix"), ws=None, cols=10, pcols=10,
                  **over) == ema.EMA_ERR_WORKSPACE
    return int(re.search(r"workspace of (\d+) bytes needed", ema.last_error()).group(1))


def test_workspace_is_enough_for_smaller_calls(ema):
    """A workspace of some bounds holds every call whose bounds are no larger."""
    rng = random.Random(2)
    for _ in range(3000):
        heads, hkv = rng.choice([(32, 8), (16, 2), (12, 1), (8, 8), (64, 8)])
        B, max_q = rng.randint(1, 200), rng.choice([1, rng.randint(1, 300)])
        n, max_len = rng.randint(B, B * max_q), rng.randint(1, 40000)
        prefix = rng.choice([0, 1, 1]) * rng.randint(1, 40000)
        size = ema.paged_workspace_size(B, n, heads, hkv, 128, max_q, max_len, prefix)
        b, q = rng.randint(1, B), rng.randint(1, max_q)
        a = dict(heads=heads, hkv=hkv, batch=b, rows=rng.randint(1, min(n, b * q)), max_q=q, max_len=rng.randint(0, max_len))
        assert needed(ema, prefix=False, **a) <= size
        if prefix:
            assert needed(ema, prefix=True, max_prefix=rng.randint(1, prefix), **a) <= size


@pytest.mark.parametrize("prefix", [False, True])
def test_a_bound_of_no_rows_counts_as_one(ema, prefix):
    """max_q 0 is a bound that any row is past: the call is planned as for max_q 1, so that the
    choice of a prefix's way, and with it the count of tiles, has the sequences in it."""
    for B in (1, 40, 1024):
        a = dict(heads=16, hkv=8, batch=B, rows=B, max_len=4096, prefix=prefix, max_prefix=40000)
        assert needed(ema, max_q=0, **a) == needed(ema, max_q=1, **a)
        size = [ema.paged_workspace_size(B, B, 16, 8, 128, q, 4096, 40000 if prefix else 0) for q in (0, 1)]
        assert size[0] == size[1]


def test_binding_checks_tensors(ema):
    """Shapes, types, layouts and devices are checked before the call (CPU tensors here: the call
    itself is never reached)."""
    import torch

    bf = torch.bfloat16
    cache = ema.PagedCache(6, 2, 16, 128, device="cpu")
    assert cache.n_pages == 6 and cache.page_size == 16 and cache.memory_bytes() == 2 * 6 * 2 * 16 * 128 * 2
    q, table = torch.zeros(3, 8, 128, dtype=bf), torch.zeros(3, 2, dtype=torch.int32)
    n = torch.ones(3, dtype=torch.int32)
    qkv, w = torch.zeros(3, 12 * 128, dtype=bf), torch.zeros(128, dtype=bf)

    def refused(f, *a, **k):
        with pytest.raises(ema.EmaError) as e:
            f(*a, **k)
        assert e.value.code in (ema.EMA_ERR_SHAPE, ema.EMA_ERR_INVALID_ARG)

    for bad in (q.float(), q[..., :64], q.transpose(0, 1), q[0]):
        refused(ema.paged_attention, bad, cache, table, n, 32)
    refused(ema.paged_attention, q, cache, table.long(), n, 32)
    refused(ema.paged_attention, q, cache, table[:2], n, 32)
    refused(ema.paged_attention, q, cache, table, n.long(), 32)
    refused(ema.paged_attention, q, cache, table, n, 32, q_starts=n)
    refused(ema.paged_attention, q, cache, table, n, 32, out=torch.zeros(3, 8, 128, dtype=bf))
    refused(ema.paged_attention, q, cache, table, n, 32, workspace=torch.zeros(4, dtype=torch.int32))
    refused(ema.prefix_attention, q, cache, table, n[:1], 16, table, n, 32)
    refused(ema.prefix_attention, q, cache, table[0], n, 16, table, n, 32)
    refused(ema.paged_append, qkv[:, :128], w, w, 1e-6, 1e6, n, 8, cache, table)
    refused(ema.paged_append, qkv, w[:64], w, 1e-6, 1e6, n, 8, cache, table)
    refused(ema.paged_append, qkv, w, w, 1e-6, 1e6, n, 8, cache, table, q_out=q[:2])
    refused(ema.paged_append, qkv, w, w, 1e-6, 1e6, n, 8, cache, table, prefix_len=n)
    refused(ema.PagedCache, 6, 2, 16, 128, k=torch.zeros(6, 2, 16, 128), v=torch.zeros(6, 2, 16, 128))
    refused(ema.PagedCache, 6, 2, 16, 128, k=torch.zeros(6, 2, 16, 128, dtype=bf), v=torch.zeros(6, 16, 2, 128, dtype=bf).transpose(1, 2))
    with pytest.raises(ValueError):
        ema.PagedCache(6, 2, 16, 128, device="cpu", dtype="int4")


def test_exponents_on_another_device_are_refused(ema):
    """FP8 pages whose exponents lie elsewhere than the codes: refused when the pool is made, since a
    call checks its tensors against the pool alone. (The meta device stands for any other.)"""
    import torch

    codes = [torch.zeros(6, 2, 16, 128, dtype=torch.uint8) for _ in range(2)]
    here, there = (torch.zeros(6, 2, 16, 2, dtype=torch.int8, device=d) for d in ("cpu", "meta"))
    for k_exp, v_exp, name in ((there, here, "k_exp"), (here, there, "v_exp"), (there, None, "k_exp"), (None, there, "v_exp")):
        with pytest.raises(ema.EmaError) as e:
            ema.PagedCache(6, 2, 16, 128, k=codes[0], v=codes[1], dtype="fp8", k_exp=k_exp, v_exp=v_exp, device="cpu")
        assert e.value.code == ema.EMA_ERR_INVALID_ARG and name in str(e.value)
    # those that the pool makes for itself lie with the codes, whatever the device of other tensors
    cache = ema.PagedCache(6, 2, 16, 128, k=codes[0], v=codes[1], dtype="fp8", device="meta")
    assert cache.k_exp.device == cache.v_exp.device == codes[0].device


def test_missing_tensors_are_refused(ema):
    """None (or what is no tensor) in the place of a tensor that a call cannot do without is the
    documented error, which names it."""
    import torch

    bf, i32 = torch.bfloat16, torch.int32
    cache = ema.PagedCache(6, 2, 16, 128, device="cpu")
    n, one = torch.ones(3, dtype=i32), torch.ones(1, dtype=i32)
    calls = {
        ema.paged_append: (dict(qkv=torch.zeros(3, 12 * 128, dtype=bf), offsets=n, table=torch.zeros(3, 2, dtype=i32)),
                           dict(q_norm_w=None, k_norm_w=None, eps=1e-6, theta=1e6, n_heads=8, cache=cache)),
        ema.paged_attention: (dict(q=torch.zeros(3, 8, 128, dtype=bf), table=torch.zeros(3, 2, dtype=i32), lengths=n),
                              dict(cache=cache, max_len=32)),
        ema.prefix_attention: (dict(q=torch.zeros(3, 8, 128, dtype=bf), table=torch.zeros(3, 2, dtype=i32), lengths=n,
                                    prefix_table=torch.zeros(2, dtype=i32), prefix_len=one),
                               dict(cache=cache, max_len=32, max_prefix=16)),
    }
    for call, (tensors, rest) in calls.items():
        for name in tensors:
            for bad in (None, [1, 2, 3]):
                with pytest.raises(ema.EmaError) as e:
                    call(**{**tensors, **rest, name: bad})
                assert e.value.code == ema.EMA_ERR_INVALID_ARG and name in str(e.value), (call.__name__, name)
        for name in ("q_starts", "q_out" if "qkv" in tensors else "workspace"):  # optional, but tensors if given
            with pytest.raises(ema.EmaError) as e:
                call(**{**tensors, **rest, name: [0, 1, 2, 3]})
            assert e.value.code == ema.EMA_ERR_INVALID_ARG and name in str(e.value), (call.__name__, name)
