"""GPU tests of the state space scan of bf16 prompts that are cut in time (the ends of the pieces, their joining, the
pieces from their start states), against float64: every form of the chunked kernel, and what the other tests of
the mixer calls do with shorter prompts, which run whole."""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
import mixer_ref as ref  # noqa: E402
import test_gpu_mixer as mixer  # noqa: E402
from test_gpu_mixer import BF, CHUNK_SHAPES, F32, ema, ints, rand, scan_case  # noqa: E402,F401

# H and the rows' weights in two bf16 parts where y reads them, the terms of the state in three
PARTS = dict(read_bits=2.0 ** -16, split_bits=2.0 ** -23)


def space(ema, lens, max_rows, H, P, N, G):
    """A workspace that shows whether it was written."""
    size = ema.ssm_workspace_size(len(lens), sum(lens), max_rows, H, P, N, G)
    return torch.full((size,), 85, dtype=torch.uint8, device="cuda")


@pytest.mark.parametrize("shape", CHUNK_SHAPES)
@pytest.mark.parametrize("lens,slots,offsets", [
    ([520, 3, 0, 129], [-1, 1, 0, 3], [5, 0, 2, 7]),       # a long sequence whose state is not kept
    ([520, 3, 0, 129], [4, 1 << 30, 0, 2], [0, 9, 2, 0]),  # one from zeros
    ([513, 640], [1, 0], [3, 3]),                          # last pieces of one row, and whole ones
])
def test_cut(ema, shape, lens, slots, offsets):
    ws = space(ema, lens, max(lens), *shape)
    scan_case(ema, BF, lens, *shape, 1000, offsets=offsets, slots=slots, n_slots=5, tail=0 if len(lens) == 2 else 2,
              max_rows=max(lens), workspace=ws, strided=shape[0] % 2 == 0, **PARTS)
    assert bool((ws != 85).any()), "not cut"


@pytest.mark.parametrize("shape", CHUNK_SHAPES)
def test_cut_where_heads_hardly_decay(ema, shape):
    """Steps near 0.003 at rates near -1: the state at the end is nearly all of its pieces' ends."""
    lens = [513, 400]
    ws = space(ema, lens, 513, *shape)
    scan_case(ema, BF, lens, *shape, 1010, offsets=[1, 1], softplus=False, bias=False, dt_scale=0.05, a_scale=1.5, workspace=ws,
              max_rows=513, **PARTS)
    assert bool((ws != 85).any()), "not cut"


@pytest.mark.parametrize("kw", [dict(D=False), dict(softplus=False), dict(limit=(0.05, 0.2)), dict(dt_scale=30.0),
                                dict(a_scale=1.0), dict(limit=(0.0, 0.0))])
def test_cut_options(ema, kw):
    lens = [600, 200]
    ws = space(ema, lens, 600, 4, 64, 128, 2)
    scan_case(ema, BF, lens, 4, 64, 128, 2, 1020, workspace=ws, max_rows=600, **PARTS, **kw)
    assert bool((ws != 85).any()), "not cut"


@pytest.mark.parametrize("what", ["x", "B", "C", "dt", "state"])
def test_values_that_are_not_finite_in_cut_prompts(ema, what):
    """They reach what the recurrence says they reach, across pieces too."""
    H, P, N, G, rows = 4, 64, 128, 2, 450
    n = 2 * rows
    a = dict(x=rand(1030, n, H, P, dtype=BF), dt=rand(1031, n, H, dtype=BF), B=rand(1032, n, G, N, dtype=BF),
             C=rand(1033, n, G, N, dtype=BF), state=rand(1034, 2, H, P, N))
    A = -torch.rand(H, generator=torch.Generator().manual_seed(1035)).cuda() - 0.5
    for at in (0, 127, 128, 449):
        for bad in (math.nan, math.inf):
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
            ws = space(ema, [rows, rows], rows, H, P, N, G)
            y = ema.ssm_scan(b["x"], b["dt"], b["B"], b["C"], A, b["state"], batch=2, max_rows=rows, workspace=ws)
            torch.cuda.synchronize()
            assert bool((ws != 85).any()), "not cut"
            same = [int((torch.isfinite(g).cpu() != torch.isfinite(w)).sum()) for g, w in ((y, want), (b["state"], want_pool))]
            assert same == [0, 0], (what, at, bad, same)


def test_captured_layer_of_a_cut_prompt(ema):
    lens = [500, 40, 2]
    layer = mixer.Layer(ema, 600)
    ws = space(ema, lens, 500, layer.H, layer.P, layer.N, layer.G)
    proj, res = layer.inputs(610, sum(lens))
    layer(proj, res, ints([0, 500, 540, 542]), ints([0, 0, 0]), ints([2, 0, 4]), 500, ws)
    assert bool((ws != 85).any()), "not cut"
    mixer.test_layer_captured(ema, lens)


@pytest.mark.parametrize("starts", [[0, 600, 20, 700], [-7, 500, 500, 1 << 30], [690, 10, 650, 0], [0, 0, 0, 700]])
def test_row_starts_that_are_no_row_starts_in_cut_calls(ema, starts):
    """They are taken as given only inside the rows: nothing outside the output, the pool and the workspace is written."""
    n, H, P, N, pad = 700, 2, 32, 64, 4096
    size = ema.ssm_workspace_size(3, n, n, H, P, N, 1)
    assert size > 0
    bufs = [torch.full((k + 2 * pad,), 3, dtype=t, device="cuda") for k, t in ((n * H * P, BF), (3 * H * P * N, F32), (size, torch.uint8))]
    y, state, ws = (b[pad:-pad] for b in bufs)
    ema.ssm_scan(rand(1040, n, H, P, dtype=BF), rand(1041, n, H, dtype=BF), rand(1042, n, 1, N, dtype=BF),
                 rand(1043, n, 1, N, dtype=BF), -torch.ones(H, device="cuda"), state.view(3, H, P, N), starts=ints(starts),
                 max_rows=n, out=y.view(n, H, P), workspace=ws)
    torch.cuda.synchronize()
    for b in bufs:
        assert bool((b[:pad] == 3).all()) and bool((b[-pad:] == 3).all())


def test_a_uniform_step_allocates_no_workspace(ema, monkeypatch):
    """Without starts the bound of a sequence's rows is known: one row of each of 512 sequences is not cut."""
    sizes, size = [], ema.ssm_workspace_size
    monkeypatch.setattr(ema, "ssm_workspace_size", lambda *a: sizes.append(size(*a)) or sizes[-1])
    B, H, P, N = 512, 2, 64, 128
    a = dict(x=rand(1050, B, H, P, dtype=BF), dt=rand(1051, B, H, dtype=BF), B=rand(1052, B, 1, N, dtype=BF),
             C=rand(1053, B, 1, N, dtype=BF), A=-torch.ones(H, device="cuda"))
    state = torch.zeros(B, H, P, N, device="cuda")
    for max_rows in (None, B, 1):
        ema.ssm_scan(**a, state=state, max_rows=max_rows)
    assert sizes == [0, 0, 0]
