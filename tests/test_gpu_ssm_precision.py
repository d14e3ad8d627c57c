"""GPU tests of how exactly the state space scan of bf16 prompts computes (ema_ssm_scan in chunks, whole and
cut in time), against float64.

An output in bf16 hides errors below 2^-8 of its value, so most of these make y small beside its terms: every
row of x is a multiple of one vector x0 and the start state is x0 times a vector, so that the scan of row t is a
number times x0 and D can be set to cancel it in one row of each head.
"""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
import mixer_ref as ref  # noqa: E402
from mixer_ref import HALF, TINY, U  # noqa: E402
from test_gpu_mixer import BF, ema, ints, rand  # noqa: E402,F401


def prompt(seed, n, H, P, N, G, dt=None, A=None, rho=None):
    """One sequence of n rows whose x is rho[t] (a power of two, or 0) times one vector a head; dt is the step."""
    x0 = rand(seed, H, P, dtype=BF, device="cpu")
    rho = torch.ones(n) if rho is None else rho
    v = rand(seed + 1, H, N, scale=0.3, device="cpu")
    g = torch.Generator().manual_seed(seed + 2)
    dt = (0.01 + 0.3 * torch.rand(n, H, generator=g)).to(BF) if dt is None else dt.to(BF)
    A = -(1 + 3 * torch.rand(H, generator=g)) if A is None else A
    return dict(x=(rho[:, None, None] * x0.float()).to(BF), dt=dt, B=rand(seed + 3, n, G, N, dtype=BF, device="cpu"),
                C=rand(seed + 4, n, G, N, dtype=BF, device="cpu"), A=A, state=(x0.float()[:, :, None] * v[:, None])[None])


def cancelling(a, rows):
    """D such that y of row rows[h] of head h is close to 0."""
    y, _, _, _ = ref.scan(*(a[k] for k in ("x", "dt", "B", "C", "A", "state")), 1, softplus=False)
    x = a["x"].double()
    return torch.stack([-(y[t, h] * x[t, h]).sum() / (x[t, h] ** 2).sum() for h, t in enumerate(rows)]).float()


def run(ema, a, D, workspace=None, max_rows=None):
    c = {k: v.cuda() for k, v in a.items()}
    y = ema.ssm_scan(**c, D=None if D is None else D.cuda(), batch=1, offsets=ints([1]), softplus=False, max_rows=max_rows,
                     workspace=workspace)
    torch.cuda.synchronize()
    return y, c["state"]


def held(ema, a, rows, read_bits, what, live=None):
    """y within its rounding, the sums' and read_bits of its terms, where the last two decide: the rows that cancel.
    live: how many rows back the terms come from that are not nothing."""
    n, N = a["x"].shape[0], a["state"].shape[3]
    live = live or n
    D = cancelling(a, rows)
    want, _, mag, _ = ref.scan(*(a[k] for k in ("x", "dt", "B", "C", "A", "state")), 1, D, softplus=False)
    near = torch.stack([want[t, h].abs() / mag[t, h] for h, t in enumerate(rows)])
    assert float(near.max()) < 2.0 ** -18, "the inputs of this test do not cancel"
    got, _ = run(ema, a, D)
    tol = HALF[BF] * want.abs() + ((2 * live + N + 16) * U + 2.0 ** -21 + read_bits) * mag + TINY[BF]
    ref.check(got, want, tol, what)


SHAPES = [(32, 32, 64, 1), (16, 64, 128, 2), (8, 128, 128, 1), (16, 64, 256, 4), (12, 96, 64, 2), (6, 160, 128, 1)]


@pytest.mark.parametrize("shape", SHAPES)
def test_skip_term_is_in_32_bits(ema, shape):
    """y is D x to the last bit where B and C are small; D lies half a step of bf16 beside its values."""
    H, P, N, G = shape
    a = prompt(10, 70, *shape)
    a["B"] = (a["B"].float() * 2.0 ** -12).to(BF)
    a["C"] = (a["C"].float() * 2.0 ** -12).to(BF)
    D = 1 + 2.0 ** -8 + 2.0 ** -7 * torch.arange(H) + 2.0 ** -20
    want, _, mag, _ = ref.scan(*(a[k] for k in ("x", "dt", "B", "C", "A", "state")), 1, D, softplus=False)
    scan = mag - (D.double()[:, None] * a["x"].double()).abs()
    got, _ = run(ema, a, D)
    # the scan's own terms are below 2^-7 of y's rounding whatever they are rounded to
    ref.check(got, want, HALF[BF] * want.abs() + 2.0 ** -7 * scan + 8 * U * mag + TINY[BF], f"skip {shape}")


# H and M each in two bf16 parts: off by at most half a step of half a step, 2^-16 of the term
PARTS = 2.0 ** -16


@pytest.mark.parametrize("shape", SHAPES)
def test_terms_of_a_prompt(ema, shape):
    """The weights of the rows and the start state where y reads them, in rows all over a chunk."""
    H = shape[0]
    a = prompt(20, 70, *shape)
    held(ema, a, [(7 * h + 3) % 70 for h in range(H)], PARTS, f"terms {shape}")
    a["state"] = torch.zeros_like(a["state"])
    held(ema, a, [(5 * h + 1) % 70 for h in range(H)], PARTS, f"rows' terms {shape}")


def test_terms_of_a_prompt_cut_in_time(ema):
    a = prompt(30, 600, 8, 64, 128, 2)
    held(ema, a, [599, 511, 512, 300, 127, 128, 200, 64], PARTS, "cut")


@pytest.mark.parametrize("shape", SHAPES)
def test_weak_decays_behind_strong_ones(ema, shape):
    """14 rows that forget everything, then two that forget little, again and again: the little is not lost in
    a sum with the other."""
    H, n = shape[0], 64
    weak = 2.0 ** -7 * (1 + torch.arange(H) / 64)
    dt = torch.where(torch.arange(n)[:, None] % 16 < 14, torch.tensor(8.0), weak)
    a = prompt(40, n, *shape, dt=dt, A=torch.full((H,), -16.0))
    held(ema, a, [16 * (h % 4) + 15 for h in range(H)], PARTS, f"strong and weak {shape}", live=3)


@pytest.mark.parametrize("rows,cut", [(100, False), (513, True), (640, True)])
@pytest.mark.parametrize("shape", [(4, 32, 64, 1), (4, 64, 128, 2), (2, 128, 256, 1), (2, 160, 128, 1)])
def test_state_of_a_prompt_keeps_32_bits(ema, rows, cut, shape):
    """Rows that are added to a state that does not decay, each to a column of its own: a step of 16 bits times a
    value of 8 is exact in 32, and stays so however a prompt is cut."""
    H, P, N, G = shape
    x = rand(50, rows, H, P, dtype=BF)
    b = torch.zeros(rows, G, N, dtype=BF, device="cuda")
    for t in range(N):
        b[(t * 131) % rows if t < rows else 0, :, t] = 1.0  # (131 has no divisor in common with the row counts)
    state = torch.zeros(1, H, P, N, device="cuda")
    step = 43691 / 32768  # 16 bits, every other one set
    bias = torch.full((H,), step, device="cuda")
    need = ema.ssm_workspace_size(1, rows, rows, H, P, N, G)
    ws = torch.full((need,), 85, dtype=torch.uint8, device="cuda")
    ema.ssm_scan(x, torch.zeros(rows, H, dtype=BF, device="cuda"), b, torch.zeros_like(b), torch.zeros(H, device="cuda"), state,
                 dt_bias=bias, softplus=False, batch=1, offsets=ints([0]), workspace=ws)
    torch.cuda.synchronize()
    assert bool((ws != 85).any()) == cut, "this test is of calls that are cut, or of calls that are not"
    want = torch.zeros(1, H, P, N, dtype=torch.float64)
    for t in range(min(N, rows)):
        want[0, :, :, t] += ref.f64(x[(t * 131) % rows]) * step
    if N > rows:  # the columns from `rows` on took row 0
        want[0, :, :, rows:] += (ref.f64(x[0]) * step)[:, :, None]
    # (step and product have at most 24 bits, each column one of them)
    assert torch.equal(state.cpu().double(), want)
