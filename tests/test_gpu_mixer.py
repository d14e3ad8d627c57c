"""GPU tests of the mixer calls (ema_causal_conv, ema_ssm_scan, ema_gated_norm, ema_residual_norm) against their
definitions in float64 (mixer_ref.py), at the sizes and layouts where they can go wrong."""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
import mixer_ref as ref  # noqa: E402
from mixer_ref import HALF, TINY, U  # noqa: E402

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
TYPES = [BF, HF, F32]


@pytest.fixture(scope="module")
def ema():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a ROCm GPU")
    import ema_attn

    ema_attn.lib()
    return ema_attn


def rand(seed, *shape, dtype=F32, scale=1.0, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(device)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def wide(t, before=8, after=8):
    """The same values as a piece of wider rows."""
    n, inner = t.shape[0], t[0].numel() if t.shape[0] else math.prod(t.shape[1:])
    w = torch.full((n, before + inner + after), 77.0, dtype=t.dtype, device=t.device)
    w[:, before:before + inner] = t.reshape(n, inner)
    return w[:, before:before + inner].unflatten(1, t.shape[1:]) if t.dim() > 2 else w[:, before:before + inner]


# ------------------------------------------------------------------ convolution
def conv_case(ema, dtype, lens, C, W, seed, *, bias=True, silu=True, state=True, offsets=None, slots=None, n_slots=None,
              tail=0, strided=False, batch=None, max_rows=None):
    n, B = sum(lens) + tail, len(lens)
    starts = ints([sum(lens[:i]) for i in range(B + 1)]) if len(set(lens)) > 1 or tail else None
    x = rand(seed, n, C, dtype=dtype)
    w = rand(seed + 1, C, W, dtype=dtype, scale=0.5)
    b = rand(seed + 2, C, dtype=dtype, scale=0.2) if bias else None
    pool = rand(seed + 3, n_slots or B, W - 1, C, dtype=dtype) if state else None
    off, sl = (None if v is None else ints(v) for v in (offsets, slots))
    want, want_pool, mag = ref.conv(x, w, b, pool, B, None if starts is None else starts.tolist(), offsets, slots, silu)
    out = torch.full((n, C), 5.0, dtype=dtype, device="cuda")
    xx, oo = (wide(x), wide(out)) if strided else (x, out)
    ema.causal_conv(xx, w, bias=b, state=pool, starts=starts, offsets=off, slots=sl, batch=B, silu=silu, out=oo,
                    max_rows=max_rows)
    torch.cuda.synchronize()
    used = sum(lens)
    assert bool((oo[used:] == 5.0).all()), "rows behind the last sequence"
    # W + 1 sums, the activation (its slope is at most 1.1) and one rounding
    tol = HALF[dtype] * want.abs() + 1.1 * (W + 1) * U * mag + 2.0 ** -21 * want.abs() + TINY[dtype]
    ref.check(oo[:used], want[:used], tol[:used], f"conv {dtype} {lens} C={C} W={W}")
    if state:
        assert torch.equal(pool.cpu().double(), want_pool), "the kept inputs are copies"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("W", [2, 3, 4])
def test_conv_lengths(ema, dtype, W):
    lens = [1, 2, 3, 4, 5, 0, 31, 32, 33, 64, 65, 97, 0]
    conv_case(ema, dtype, lens, 520, W, 10, offsets=[5, 0, 7, 1, 0, 3, 1, 0, 1, 1, 0, 9, 0], n_slots=20,
              slots=[19, 3, 4, 0, 1, 2, 8, 9, 10, 11, 12, 13, 14], tail=5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("C", [1, 7, 8, 512, 1031, 8192])
def test_conv_channels_and_strides(ema, dtype, C):
    conv_case(ema, dtype, [1, 40], C, 4, 20, bias=C != 8, silu=C != 7, strided=C != 1)
    conv_case(ema, dtype, [1] * 9, C, 4, 21, strided=True)
    conv_case(ema, dtype, [3], C, 2, 22, state=False)


def test_conv_slots_that_are_not_there(ema):
    """A slot outside the pool is not followed: zeros before the sequence, nothing kept."""
    conv_case(ema, BF, [2, 5, 40, 1], 64, 4, 30, slots=[-1, 3, 1 << 30, 2], n_slots=5, offsets=[4, 4, 4, 4])


def test_conv_many_sequences(ema):
    lens = [(i * 7) % 5 for i in range(700)]
    conv_case(ema, BF, lens, 16, 4, 40, offsets=[i % 3 for i in range(700)])
    conv_case(ema, F32, [1] * 4096, 4, 3, 41)


def test_conv_of_pieces_is_the_conv_of_the_whole(ema):
    """A prompt in chunks and single tokens: the same bits as at once."""
    C, W, n = 264, 4, 150
    x, w, b = rand(50, n, C, dtype=BF), rand(51, C, W, dtype=BF), rand(52, C, dtype=BF)
    pool = rand(53, 2, W - 1, C, dtype=BF)
    whole = ema.causal_conv(x, w, bias=b, state=pool, offsets=ints([0]), slots=ints([1]))
    kept = pool.clone()
    pool2 = rand(53, 2, W - 1, C, dtype=BF)
    at, got = 0, []
    for n_i in [1, 1, 2, 60, 3, 1, 82]:
        got.append(ema.causal_conv(x[at:at + n_i], w, bias=b, state=pool2, offsets=ints([at]), slots=ints([1])))
        at += n_i
    assert torch.equal(torch.cat(got), whole) and torch.equal(pool2, kept)


def test_conv_values_that_are_not_finite_stay_in_their_channel(ema):
    x, w = rand(60, 40, 64, dtype=BF), rand(61, 64, 4, dtype=BF)
    clean = ema.causal_conv(x, w, batch=1)
    x[7, 3], x[20, 10] = math.nan, math.inf
    got = ema.causal_conv(x, w, batch=1)
    touched = torch.zeros(40, 64, dtype=torch.bool, device="cuda")
    touched[7:11, 3], touched[20:24, 10] = True, True
    assert torch.equal(got[~touched], clean[~touched]) and bool(got[7:11, 3].isnan().all())


# ------------------------------------------------------------------ scan
def scan_case(ema, dtype, lens, H, P, N, G, seed, *, offsets=None, slots=None, n_slots=None, tail=0, strided=False,
              D=True, bias=True, softplus=True, limit=(0.0, math.inf), max_rows=None, a_scale=16.0, workspace=None,
              split_bits=0.0, dt_scale=1.0, read_bits=0.0):
    n, B = sum(lens) + tail, len(lens)
    starts = ints([sum(lens[:i]) for i in range(B + 1)]) if len(set(lens)) > 1 or tail else None
    x = rand(seed, n, H, P, dtype=dtype)
    bm, cm = rand(seed + 1, n, G, N, dtype=dtype), rand(seed + 2, n, G, N, dtype=dtype)
    dt = rand(seed + 3, n, H, dtype=dtype, scale=dt_scale)
    if not softplus:
        dt = dt.abs() * 0.1
    A = -(1 + (a_scale - 1) * torch.rand(H, generator=torch.Generator().manual_seed(seed + 4))).cuda()
    Dw = rand(seed + 5, H) if D else None
    db = (rand(seed + 6, H) - 3) if bias else None
    state = rand(seed + 7, n_slots or B, H, P, N, scale=0.3)
    off, sl = (None if v is None else ints(v) for v in (offsets, slots))
    want, want_pool, mag, pool_mag = ref.scan(x, dt, bm, cm, A, state, B, Dw, db,
                                              None if starts is None else starts.tolist(), offsets, slots, softplus, limit)
    out = torch.full((n, H, P), 5.0, dtype=dtype, device="cuda")
    xx, oo, bb, cc, tt = (wide(t, 8, 16) for t in (x, out, bm, cm, dt)) if strided else (x, out, bm, cm, dt)
    untouched = state.clone()
    ema.ssm_scan(xx, tt, bb, cc, A, state, D=Dw, dt_bias=db, starts=starts, offsets=off, slots=sl, batch=B,
                 max_rows=max_rows, softplus=softplus, dt_limit=limit, out=oo, workspace=workspace)
    torch.cuda.synchronize()
    used = sum(lens)
    assert bool((oo[used:] == 5.0).all()), "rows behind the last sequence"
    # every row's step adds a few roundings of the state, the sums over rows and d_state theirs
    rows = max(lens) if lens else 0
    tol_y = HALF[dtype] * want.abs() + ((2 * rows + N + 16) * U + 2.0 ** -21 + read_bits) * mag + TINY[dtype]
    tol_s = ((2 * rows + 16) * U + 2.0 ** -21 + split_bits) * pool_mag + 1e-37
    ref.check(oo[:used], want[:used], tol_y[:used], f"scan {dtype} {lens[:12]} H={H} P={P} N={N} G={G}: y")
    ref.check(state, want_pool, tol_s, "  state")
    held = set(range(B)) if slots is None else {s for s, l in zip(slots, lens) if l}
    for i in range(state.shape[0]):
        if i not in held or (slots is None and lens[i] == 0):
            assert torch.equal(state[i], untouched[i]), "a slot that no sequence has"


SHAPES = [(4, 64, 128, 2), (3, 48, 80, 3), (8, 32, 64, 1), (2, 128, 256, 2), (5, 20, 36, 1), (2, 1, 4, 1), (1, 65, 16, 1)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_scan_tokens(ema, dtype, shape):
    scan_case(ema, dtype, [1] * 5, *shape, 100, slots=[6, 0, 3, -1, 5], n_slots=7, offsets=[3, 0, 1, 2, 8])
    scan_case(ema, dtype, [1, 0, 3, 7, 2], *shape, 101, strided=shape[0] % 2 == 0, tail=3, max_rows=1)


@pytest.mark.parametrize("dtype", [HF, F32])
@pytest.mark.parametrize("shape", SHAPES)
def test_scan_prompts(ema, dtype, shape):
    scan_case(ema, dtype, [1, 0, 33, 64, 130, 31], *shape, 110, slots=[6, 0, 3, 2, 5, 1], n_slots=7,
              offsets=[3, 0, 1, 0, 8, 0], tail=2)


# in chunks on the matrix cores: H and M are rounded to bf16 where y reads them, the terms of the state to two
CHUNKED = dict(read_bits=2.0 ** -8, split_bits=2.0 ** -16)
CHUNK_SHAPES = [(4, 64, 128, 2), (3, 64, 64, 1), (4, 32, 64, 1), (5, 32, 128, 1), (2, 96, 128, 1), (2, 128, 256, 1),
                (1, 160, 128, 1), (8, 64, 128, 8)]


@pytest.mark.parametrize("shape", CHUNK_SHAPES)
def test_scan_chunks(ema, shape):
    scan_case(ema, BF, [1, 0, 33, 64, 130, 31], *shape, 140, slots=[6, 0, 3, 2, 5, 1], n_slots=7,
              offsets=[3, 0, 1, 0, 8, 0], tail=2, **CHUNKED)
    scan_case(ema, BF, [65, 65], *shape, 141, strided=True, slots=[-1, 1], n_slots=2, **CHUNKED)


@pytest.mark.parametrize("dtype,extra", [(BF, CHUNKED), (F32, {})])
def test_scan_in_pieces(ema, dtype, extra):
    """Few heads and long sequences: cut in time, with as much workspace as they like, some, and none."""
    lens = [700, 3, 0, 257]
    need = ema.ssm_workspace_size(4, sum(lens), 700, 2, 64, 128, 1, dtype)
    assert need > 0
    for size in [need, need // 2, need // 4, 16, 0]:
        ws = torch.empty(size, dtype=torch.uint8, device="cuda")
        scan_case(ema, dtype, lens, 2, 64, 128, 1, 150, offsets=[5, 0, 2, 0], workspace=ws, max_rows=700, a_scale=1.5,
                  **extra)
    # bounds below the true lengths: another way, the same result
    scan_case(ema, dtype, lens, 2, 64, 128, 1, 150, offsets=[5, 0, 2, 0], max_rows=1, a_scale=1.5)
    scan_case(ema, dtype, lens, 2, 64, 128, 1, 150, offsets=[5, 0, 2, 0], max_rows=130, a_scale=1.5, **extra)


def test_scan_chunk_options(ema):
    for i, kw in enumerate([dict(D=False), dict(bias=False), dict(softplus=False), dict(limit=(0.05, 0.2)),
                            dict(dt_scale=30.0), dict(a_scale=1.0), dict(limit=(0.0, 0.0)), dict(limit=(5.0, math.inf))]):
        scan_case(ema, BF, [100, 40], 4, 64, 128, 2, 160 + i, **CHUNKED, **kw)


@pytest.mark.parametrize("what", ["x", "B", "C", "dt", "state"])
@pytest.mark.parametrize("rows", [1, 100])
def test_scan_values_that_are_not_finite(ema, what, rows):
    """They reach what the recurrence says they reach: no earlier row, no other column, head or sequence."""
    H, P, N, G = 4, 64, 128, 2
    n = 2 * rows
    a = dict(x=rand(170, n, H, P, dtype=BF), dt=rand(171, n, H, dtype=BF), B=rand(172, n, G, N, dtype=BF),
             C=rand(173, n, G, N, dtype=BF), state=rand(174, 2, H, P, N))
    A = -torch.rand(H, device="cuda") - 0.5
    at = rows // 2
    for bad in (math.nan, math.inf, -math.inf):
        b = {k: v.clone() for k, v in a.items()}
        if what == "state":
            b["state"][0, 1, 5, 7] = bad
        elif what == "x":
            b["x"][at, 1, 5] = bad
        elif what == "dt":
            b["dt"][at, 1] = math.nan
        else:
            b[what][at, 1, 7] = bad
        want, want_pool, _, _ = ref.scan(b["x"], b["dt"], b["B"], b["C"], A, b["state"], 2)
        y = ema.ssm_scan(b["x"], b["dt"], b["B"], b["C"], A, b["state"], batch=2)
        torch.cuda.synchronize()
        same = [int((torch.isfinite(g).cpu() != torch.isfinite(w)).sum()) for g, w in ((y, want), (b["state"], want_pool))]
        assert same == [0, 0], (what, bad, same)


@pytest.mark.parametrize("rows", [3, 100])
def test_scan_decay_rates_not_finite(ema, rows):
    """A head whose rate is NaN has no finite value; one of -inf forgets all but the row itself."""
    H, P, N, n = 4, 32, 64, 2 * rows
    x, b, c = rand(180, n, H, P, dtype=BF), rand(181, n, 1, N, dtype=BF), rand(182, n, 1, N, dtype=BF)
    dt, state = rand(183, n, H, dtype=BF), rand(184, 2, H, P, N)
    A = torch.tensor([-1.0, math.nan, -math.inf, 0.0], device="cuda")
    want, pool, mag, pool_mag = ref.scan(x, dt, b, c, torch.where(A == -math.inf, -1e30, A), state, 2)
    y = ema.ssm_scan(x, dt, b, c, A, state, batch=2)
    for got, w, m, half in ((y, want, mag, HALF[BF]), (state, pool, pool_mag, 0.0)):
        assert bool(torch.isnan(got[:, 1]).all())
        keep = [0, 2, 3]
        # (H and the weights of a chunk, rounded to bf16 as operands of y, and y itself)
        ref.check(got[:, keep], w[:, keep], (3 * half + (2 * rows + N + 96) * U) * m[:, keep] + TINY[BF], "kept heads")


def test_scan_options(ema):
    for i, kw in enumerate([dict(D=False), dict(bias=False), dict(softplus=False), dict(limit=(0.05, 0.2)),
                            dict(dt_scale=30.0), dict(a_scale=1.0)]):
        scan_case(ema, F32, [40, 3], 4, 64, 128, 2, 120 + i, **kw)


def test_scan_many_sequences(ema):
    scan_case(ema, F32, [(i * 7) % 4 for i in range(300)], 2, 16, 16, 1, 130, offsets=[i % 3 for i in range(300)])


# How many state rows a lane holds goes by the waves that there are: sequences (whole) and long ones (cut in
# time) that take two and four of them, of sizes that fill the lanes and that do not.
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,shape", [(10, (8, 64, 64, 2)), (33, (16, 64, 64, 1)), (22, (8, 40, 36, 2)), (44, (16, 40, 36, 4)),
                                         (9, (16, 64, 256, 1)), (33, (16, 64, 132, 2))])
def test_scan_lanes_whole(ema, dtype, batch, shape):
    scan_case(ema, dtype, [(3 * i) % 11 for i in range(batch)], *shape, 140, max_rows=31, strided=batch % 2 == 0)


@pytest.mark.parametrize("dtype", [HF, F32])
@pytest.mark.parametrize("rows,shape", [(300, (32, 64, 64, 2)), (300, (64, 64, 64, 1)), (250, (32, 40, 36, 2)),
                                        (360, (64, 40, 36, 4))])
def test_scan_lanes_cut(ema, dtype, rows, shape):
    H, P, N, G = shape
    assert ema.ssm_workspace_size(2, rows + 5, rows, H, P, N, G, dtype) > 0
    scan_case(ema, dtype, [rows, 5], *shape, 150, offsets=[7, 0], tail=2)


# ------------------------------------------------------------------ gated norm
def gated_case(ema, dtype, n, dim, group, seed, *, gate=True, first=False, sigmoid=False, unit=False, w="dim",
               strided=False, scale=1.0, inplace=False):
    x = rand(seed, n, dim, dtype=dtype, scale=scale)
    z = rand(seed + 1, n, dim, dtype=dtype) if gate else None
    wt = None if w is None else (rand(seed + 2, group if w == "group" else dim, scale=0.2) + (0 if unit else 1)).to(dtype)
    want = ref.gated(x, z, wt, 1e-5, group, first, sigmoid, unit)
    out = torch.empty_like(x)
    if strided:
        x, out = wide(x), wide(out)
        z = None if z is None else wide(z, 16, 8)
    got = ema.gated_norm(x, z, wt, 1e-5, group=group, gate_first=first, sigmoid=sigmoid, unit_offset=unit,
                         out=x if inplace else out)
    torch.cuda.synchronize()
    # the sum of squares (at most group + 8 steps, half of which reaches the root) and the factors
    tol = (HALF[dtype] + (group + 8) * U + 2.0 ** -20) * want.abs() + TINY[dtype]
    ref.check(got, want, tol, f"gated {dtype} [{n}, {dim}/{group}]")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,group", [(128, 128), (1024, 64), (1000, 40), (1536, 192), (1024, 512), (99, 33), (520, 520),
                                       (3000, 1500), (4096, 4096), (2049, 2049), (8192, 8192), (16384, 16384), (9001, 9001),
                                       (7, 1), (5, 5)])
def test_gated_sizes(ema, dtype, dim, group):
    gated_case(ema, dtype, 3, dim, group, 200)
    gated_case(ema, dtype, 5, dim, group, 201, first=True, w="group", strided=True)


@pytest.mark.parametrize("kw", [dict(gate=False), dict(sigmoid=True), dict(first=True, sigmoid=True), dict(unit=True),
                                dict(w=None), dict(w=None, gate=False), dict(unit=True, w="group"), dict(inplace=True),
                                dict(inplace=True, strided=True), dict(scale=1e-3), dict(scale=1e3)])
@pytest.mark.parametrize("group", [128, 640])
def test_gated_options(ema, kw, group):
    gated_case(ema, BF, 65, 640, group, 210, **kw)


def test_gated_zero_rows_and_no_rows(ema):
    x = torch.zeros(2, 256, dtype=BF, device="cuda")
    z, w = rand(220, 2, 256, dtype=BF), rand(221, 256, dtype=BF)
    assert bool((ema.gated_norm(x, z, w, 1e-6) == 0).all())
    assert ema.gated_norm(x[:0], z[:0], w, 1e-6).shape == (0, 256)


# ------------------------------------------------------------------ residual norm
def residual_case(ema, dtype, n, dim, seed, *, stream=None, post=True, gate=None, scale=0.7, unit=False, pre=True,
                  strided=False, inplace=False):
    stream = stream or dtype
    br, res = rand(seed, n, dim, dtype=dtype), rand(seed + 1, n, dim, dtype=stream)
    pw = (rand(seed + 2, dim, scale=0.2) + (0 if unit else 1)).to(dtype) if pre else None
    qw = (rand(seed + 3, dim, scale=0.2) + (0 if unit else 1)).to(dtype) if post else None
    g = None if gate is None else rand(seed + 4, *((dim,) if gate == "one" else (n, dim)), dtype=dtype)
    h, want, mag = ref.residual(br, res, pw, 1e-5, qw, g, scale, unit)
    out = torch.empty_like(br) if pre else None
    if strided:
        br, res, out = wide(br), wide(res), wide(out) if pre else None
        g = wide(g, 16, 8) if gate == "rows" else g
    got = ema.residual_norm(br, res, pw, 1e-5, post_weight=qw, gate=g, scale=scale, unit_offset=unit,
                            out=br if inplace else out)
    torch.cuda.synchronize()
    each = ((dim + 8) * U + 2.0 ** -20) * mag  # of h: the branch's norm, its factors, the sum
    ref.check(res, h, HALF[stream] * h.abs() + each + TINY[stream], f"residual {dtype}/{stream} [{n}, {dim}]: h")
    if pre:
        root = torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-5)
        w = ref.f64(pw).abs() if not unit else (1 + ref.f64(pw)).abs()
        # what h is off by, in each value and in the root, beside the roundings of the norm itself
        off = each / root * w + (each * h.abs()).mean(-1, keepdim=True) / root ** 2 * want.abs()
        ref.check(got, want, (HALF[dtype] + (dim + 8) * U + 2.0 ** -20) * want.abs() + off + TINY[dtype], "  out")
    else:
        assert got is None


@pytest.mark.parametrize("dtype,stream", [(BF, BF), (BF, F32), (HF, HF), (HF, F32), (F32, F32)])
@pytest.mark.parametrize("dim", [1, 8, 100, 512, 1111, 2048, 4096, 5120, 8192, 9001, 16384])
def test_residual_sizes(ema, dtype, stream, dim):
    residual_case(ema, dtype, 3, dim, 300, stream=stream, gate="rows")
    residual_case(ema, dtype, 2, dim, 301, stream=stream, post=False, strided=True, gate="one")


@pytest.mark.parametrize("kw", [dict(), dict(post=False), dict(unit=True), dict(pre=False), dict(gate="one"), dict(gate="rows"),
                                dict(inplace=True), dict(inplace=True, strided=True), dict(scale=-2.0), dict(scale=0.0)])
def test_residual_options(ema, kw):
    residual_case(ema, BF, 33, 768, 310, **kw)
    residual_case(ema, BF, 33, 768, 311, stream=F32, **kw)


# ------------------------------------------------------------------ together
class Layer:
    """A recurrent mixer layer between two norms, as a server runs it: the projections' outputs come in."""

    def __init__(self, ema, seed, dtype=BF, n_slots=5, H=8, P=64, G=2, N=128):
        self.ema, self.H, self.P, self.G, self.N, self.dtype = ema, H, P, G, N, dtype
        self.inner, self.conv_dim = H * P, H * P + 2 * G * N
        self.cw, self.cb = rand(seed, self.conv_dim, 4, dtype=dtype, scale=0.5), rand(seed + 1, self.conv_dim, dtype=dtype, scale=0.1)
        self.A = -(0.5 + 4 * torch.rand(H, generator=torch.Generator().manual_seed(seed + 2))).cuda()
        self.D, self.dt_bias = rand(seed + 3, H), rand(seed + 4, H) - 3
        self.gw = (1 + rand(seed + 5, self.inner, scale=0.1)).to(dtype)
        self.pre = (1 + rand(seed + 6, self.inner, scale=0.1)).to(dtype)
        self.post = (1 + rand(seed + 7, self.inner, scale=0.1)).to(dtype)
        # what a fresh slot holds does not matter
        self.conv_state = torch.full((n_slots, 3, self.conv_dim), math.nan, dtype=dtype, device="cuda")
        self.ssm_state = torch.full((n_slots, H, P, N), math.nan, device="cuda")

    def __call__(self, proj, residual, starts=None, offsets=None, slots=None, max_rows=None, workspace=None, stream=None):
        """proj: [z | x B C | dt] rows of the in projection. Returns the normed rows for the next block."""
        e, H, P, G, N, I = self.ema, self.H, self.P, self.G, self.N, self.inner
        seq = dict(starts=starts, offsets=offsets, slots=slots, max_rows=max_rows, stream=stream)
        xbc = e.causal_conv(proj[:, I:I + self.conv_dim], self.cw, bias=self.cb, state=self.conv_state, **seq)
        y = e.ssm_scan(xbc[:, :I].unflatten(1, (H, P)), proj[:, I + self.conv_dim:I + self.conv_dim + H],
                       xbc[:, I:I + G * N].unflatten(1, (G, N)), xbc[:, I + G * N:].unflatten(1, (G, N)), self.A,
                       self.ssm_state, D=self.D, dt_bias=self.dt_bias, workspace=workspace, **seq).flatten(1)
        e.gated_norm(y, proj[:, :I], self.gw, 1e-5, group=I // G, gate_first=True, out=y, stream=stream)
        return e.residual_norm(y, residual, self.pre, 1e-5, post_weight=self.post, scale=0.5, out=y, stream=stream)

    def exact(self, proj, residual):
        """The same for one sequence from its start, in float64."""
        H, P, G, N, I, n = self.H, self.P, self.G, self.N, self.inner, proj.shape[0]
        p = ref.f64(proj)
        xbc, _, _ = ref.conv(p[:, I:I + self.conv_dim], self.cw, self.cb, None, 1)
        y, _, _, _ = ref.scan(xbc[:, :I].view(n, H, P), p[:, I + self.conv_dim:I + self.conv_dim + H],
                              xbc[:, I:I + G * N].view(n, G, N), xbc[:, I + G * N:].view(n, G, N), self.A,
                              torch.zeros(1, H, P, N), 1, self.D, self.dt_bias)
        y = ref.gated(y.flatten(1), p[:, :I], self.gw, 1e-5, I // G, first=True)
        h, out, _ = ref.residual(y, residual, self.pre, 1e-5, self.post, None, 0.5)
        return out, h

    def inputs(self, seed, n):
        width = self.inner + self.conv_dim + self.H
        return rand(seed, n, width + (-width) % 8, dtype=self.dtype), rand(seed + 1, n, self.inner)


# An intermediate tensor is rounded once where the definition in 64 bits has none: conv, scan, gated norm and out,
# four half steps in a row, each of which a norm or the scan's sums hand on at about its own size.
def close(got, want, dtype, what):
    g = got.detach().cpu().double()
    rel = float((g - want).norm() / want.norm())
    print(f"  {what}: relative error {rel:.3e}", flush=True)
    assert rel <= 4 * HALF[dtype], what


@pytest.mark.parametrize("dtype", TYPES)
def test_layer_prompt_then_tokens(ema, dtype):
    """Three users: prompts taken in together, in chunks, then tokens one by one, against each whole sequence."""
    layer = Layer(ema, 500, dtype)
    lens, new = [200, 33, 1], 6
    data = [layer.inputs(510 + 10 * b, n + new) for b, n in enumerate(lens)]
    outs = [[] for _ in lens]
    at = [0, 0, 0]
    slots = ints([3, 0, 4])
    for step in [[150, 33, 1], [50, 0, 0]] + [[1, 1, 1]] * new:
        rows = [(b, at[b], n) for b, n in enumerate(step)]
        proj = torch.cat([data[b][0][a:a + n] for b, a, n in rows])
        res = torch.cat([data[b][1][a:a + n] for b, a, n in rows])
        starts = ints([sum(step[:i]) for i in range(len(step) + 1)])
        out = layer(proj, res, starts=starts, offsets=ints(at), slots=slots, max_rows=max(step))
        o = 0
        for b, _, n in rows:
            outs[b].append(out[o:o + n])
            at[b] += n
            o += n
    for b in range(len(lens)):
        want, _ = layer.exact(*data[b])
        close(torch.cat(outs[b]), want, dtype, f"user {b}, {lens[b]} + {new} rows, {dtype}")


@pytest.mark.parametrize("lens", [[1, 1, 1], [300, 40, 2]])
def test_layer_captured(ema, lens):
    """A layer's step in a HIP graph, replayed with eager work of the same buffers between: every replay is
    what the eager calls give."""
    layer, n = Layer(ema, 600), sum(lens)
    starts, slots = ints([sum(lens[:i]) for i in range(len(lens) + 1)]), ints([2, 0, 4])
    offsets = ints([0, 0, 0])
    proj, res0 = layer.inputs(610, n)
    res = res0.clone()
    ws = ema.ssm_workspace(3, n, max(lens), layer.H, layer.P, layer.N, layer.G)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(proj, res, starts, offsets, slots, max(lens), ws)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(proj, res, starts, offsets, slots, max(lens), ws)
    eager = Layer(ema, 600)
    for k in range(4):
        proj.copy_(layer.inputs(620 + 10 * k, n)[0])
        res.copy_(res0)
        offsets.fill_(0 if k == 0 else 100 * k)
        graph.replay()
        torch.cuda.synchronize()
        want_res = res0.clone()
        want = eager(proj, want_res, starts, offsets, slots, max(lens), ws)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(res, want_res), k
        for a, b in ((layer.conv_state, eager.conv_state), (layer.ssm_state, eager.ssm_state)):
            assert torch.equal(a[slots.long()], b[slots.long()]), k


def test_layers_on_two_streams(ema):
    """Two users' layers on streams of their own, a workspace each, at once: what one after the other gives."""
    lens, layers = [900], [Layer(ema, 700), Layer(ema, 710)]
    data = [l.inputs(720 + 10 * i, lens[0]) for i, l in enumerate(layers)]
    want = []
    for l, (p, r) in zip(layers, data):
        want.append(l(p, r.clone(), offsets=ints([0]), slots=ints([1]), max_rows=900))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in layers]
    spaces = [ema.ssm_workspace(1, 900, 900, 8, 64, 128, 2) for _ in layers]
    zero, one = ints([0]), ints([1])
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        res = [r.clone() for _, r in data]
        torch.cuda.synchronize()
        for i, l in enumerate(layers):
            got.append(l(data[i][0], res[i], offsets=zero, slots=one, max_rows=900, workspace=spaces[i], stream=streams[i]))
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_gdn_layer(ema):
    """The pieces around the Gated DeltaNet scan: convolution of q|k|v, scan, norm of each value head, gate."""
    Hk, Hv, Dk, Dv, T = 2, 4, 128, 128, 70
    C = 2 * Hk * Dk + Hv * Dv
    qkv, w = rand(800, T, C, dtype=BF), rand(801, C, 4, dtype=BF, scale=0.5)
    z, gw = rand(802, T, Hv * Dv, dtype=BF), (1 + rand(803, Dv, scale=0.1)).to(BF)
    conv = ema.causal_conv(qkv, w, batch=1)
    q, k, v = conv.split([Hk * Dk, Hk * Dk, Hv * Dv], 1)
    # queries and keys of each head to length 1: the gated norm without gate or weight, scaled
    q = (ema.gated_norm(q, None, None, 1e-6, group=Dk).float() / Dk).to(BF)
    k = (ema.gated_norm(k, None, None, 1e-6, group=Dk).float() / math.sqrt(Dk)).to(BF)
    g = torch.sigmoid(rand(804, 1, T, Hv) + 3)
    beta = torch.sigmoid(rand(805, 1, T, Hv))
    state = torch.zeros(1, Hv, Dv, Dk, device="cuda")
    y = ema.gdn_scan(q.view(1, T, Hk, Dk), k.view(1, T, Hk, Dk), v.reshape(1, T, Hv, Dv), g, beta, state)
    out = ema.gated_norm(y.view(T, Hv * Dv), z, gw, 1e-6, group=Dv)
    torch.cuda.synchronize()
    # the definitions on the kernels' own intermediate tensors: each call within its bound
    want, _, mag = ref.conv(qkv, w, None, None, 1)
    ref.check(conv, want, HALF[BF] * want.abs() + 5.5 * U * mag + 2.0 ** -21 * want.abs() + TINY[BF], "q|k|v")
    want = ref.gated(y.view(T, Hv * Dv), z, gw, 1e-6, Dv)
    ref.check(out, want, (HALF[BF] + 136 * U + 2.0 ** -20) * want.abs() + TINY[BF], "gated heads")


# ------------------------------------------------------------------ what the header allows beyond ordinary calls
def far(t, ld):
    """The same values in rows ld elements apart."""
    n = t.shape[0]
    buf = torch.empty((n - 1) * ld + t[0].numel(), dtype=t.dtype, device="cuda")
    view = buf.as_strided((n, *t.shape[1:]), (ld, *t.stride()[1:]))
    view.copy_(t)
    return view


@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_beyond_32_bit_offsets(ema, dtype):
    """Row strides of 4 million elements: the last rows lie past 2^31 elements and 2^32 bytes."""
    n, ld = 600, 4_000_000
    C = 64
    x, w = rand(900, n, C, dtype=dtype), rand(901, C, 4, dtype=dtype)
    near, out = ema.causal_conv(x, w, batch=1), far(torch.zeros_like(x), ld)
    ema.causal_conv(far(x, ld), w, batch=1, out=out)
    assert torch.equal(out, near)
    z, gw = rand(902, n, C, dtype=dtype), rand(903, C, dtype=dtype)
    for group in (16, 64):
        ema.gated_norm(far(x, ld), far(z, ld), gw, 1e-6, group=group, out=out)
        assert torch.equal(out, ema.gated_norm(x, z, gw, 1e-6, group=group))
    res, far_res = rand(904, n, C), far(rand(904, n, C), ld)
    near = ema.residual_norm(x, res, gw, 1e-6, gate=z)
    ema.residual_norm(far(x, ld), far_res, gw, 1e-6, gate=far(z, ld), out=out)
    assert torch.equal(out, near) and torch.equal(far_res, res)
    del out, far_res
    H, P, N, G = 2, 64, 64, 1
    x, b, c = rand(905, n, H, P, dtype=dtype), rand(906, n, G, N, dtype=dtype), rand(907, n, G, N, dtype=dtype)
    dt, A = rand(908, n, H, dtype=dtype), -torch.rand(H, device="cuda") - 0.1
    s1, s2 = torch.zeros(1, H, P, N, device="cuda"), torch.zeros(1, H, P, N, device="cuda")
    near, out = ema.ssm_scan(x, dt, b, c, A, s1), far(torch.zeros_like(x), ld)
    ema.ssm_scan(far(x, ld), far(dt, ld), far(b, ld), far(c, ld), A, s2, out=out)
    assert torch.equal(out, near) and torch.equal(s1, s2)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_at_any_element(ema, dtype):
    """Rows that begin at odd elements (b and c of the scan at a multiple of four)."""
    x, w, z = rand(910, 70, 64, dtype=dtype), rand(911, 64, 4, dtype=dtype), rand(912, 70, 64, dtype=dtype)
    out = wide(torch.zeros_like(x), 3, 2)
    ema.causal_conv(wide(x, 1, 2), w, batch=1, out=out)
    assert torch.equal(out, ema.causal_conv(x, w, batch=1))
    for group in (16, 64):
        ema.gated_norm(wide(x, 1, 2), wide(z, 5, 1), None, 1e-6, group=group, out=out)
        near = ema.gated_norm(x, z, None, 1e-6, group=group)
        # (the sums of squares in another order)
        ref.check(out, near.double().cpu(), (2 * HALF[dtype] + 64 * U) * near.double().cpu().abs() + TINY[dtype], "gated")
    H, P, N, G = 2, 32, 64, 1
    x, b, c = rand(913, 70, H, P, dtype=dtype), rand(914, 70, G, N, dtype=dtype), rand(915, 70, G, N, dtype=dtype)
    dt, A = rand(916, 70, H, dtype=dtype), -torch.rand(H, device="cuda") - 0.1
    state, out = torch.zeros(1, H, P, N, device="cuda"), wide(torch.zeros_like(x), 3, 2)
    ema.ssm_scan(wide(x, 1, 2), wide(dt, 1, 2), wide(b, 4, 8), wide(c, 4, 8), A, state, out=out)
    want, pool, mag, pool_mag = ref.scan(x, dt, b, c, A, torch.zeros(1, H, P, N), 1)
    ref.check(out, want, HALF[dtype] * want.abs() + (2 * 70 + N + 32) * U * mag + TINY[dtype], "scan")
    ref.check(state, pool, (2 * 70 + 32) * U * pool_mag + 1e-37, "  state")


@pytest.mark.parametrize("starts", [[0, 50, 20, 80], [-7, 30, 30, 1000], [90, 10, 5, 0], [5, 5, 60, 70]])
def test_row_starts_that_are_no_row_starts(ema, starts):
    """They are taken as given only inside the rows: nothing outside the outputs and the slots is written."""
    n, H, P, N, C = 100, 2, 32, 64, 64
    pad = 4096

    def guarded(*shape, dtype):
        size = math.prod(shape)
        buf = torch.full((size + 2 * pad,), 3.0, dtype=dtype, device="cuda")
        return buf, buf[pad:pad + size].view(shape)

    s = ints(starts)
    ybuf, y = guarded(n, C, dtype=BF)
    pbuf, pool = guarded(3, 3, C, dtype=BF)
    ema.causal_conv(rand(920, n, C, dtype=BF), rand(921, C, 4, dtype=BF), state=pool, starts=s, out=y)
    obuf, out = guarded(n, H, P, dtype=BF)
    sbuf, state = guarded(3, H, P, N, dtype=F32)
    for max_rows in (1, n):
        ema.ssm_scan(rand(922, n, H, P, dtype=BF), rand(923, n, H, dtype=BF), rand(924, n, 1, N, dtype=BF),
                     rand(925, n, 1, N, dtype=BF), -torch.ones(H, device="cuda"), state, starts=s, max_rows=max_rows, out=out)
    torch.cuda.synchronize()
    for buf in (ybuf, pbuf, obuf, sbuf):
        assert bool((buf[:pad] == 3.0).all()) and bool((buf[-pad:] == 3.0).all())


def test_workspace_holds_what_it_says(ema):
    """The scan writes no byte behind the workspace it is told it has, whatever its size."""
    lens, H, P, N = [500, 90], 2, 64, 128
    n, pad = sum(lens), 4096
    need = ema.ssm_workspace_size(2, n, 500, H, P, N, 1)
    a = dict(x=rand(930, n, H, P, dtype=BF), dt=rand(931, n, H, dtype=BF), B=rand(932, n, 1, N, dtype=BF),
             C=rand(933, n, 1, N, dtype=BF), A=-torch.ones(H, device="cuda"))
    outs = []
    for size in (need, need - 16, need // 2, 0):
        buf = torch.full((size + pad,), 7, dtype=torch.uint8, device="cuda")
        state = torch.zeros(2, H, P, N, device="cuda")
        y = ema.ssm_scan(**a, state=state, starts=ints([0, 500, 590]), max_rows=500, workspace=buf[:size])
        torch.cuda.synchronize()
        assert bool((buf[size:] == 7).all()), size
        outs.append((y.double(), state.double()))
    for y, state in outs[1:]:
        assert float((y - outs[0][0]).norm() / outs[0][0].norm()) < 2 * HALF[BF]
        assert float((state - outs[0][1]).norm() / outs[0][1].norm()) < 1e-5
