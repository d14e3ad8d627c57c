"""The mixer calls without a GPU: their integer parts (tests/cpp/test_packed.cpp) and the calls that are refused
on the host, before any HIP call, with the documented codes."""
import ctypes
import os
import subprocess

import pytest

CPP = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp")
P = 0x40000  # an aligned address that no refused call touches
NAN, INF = float("nan"), float("inf")


def test_integer_parts():
    subprocess.run(["make", "-s", "-C", CPP, "test_packed"], check=True)
    r = subprocess.run([os.path.join(CPP, "test_packed")], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "checks passed" in r.stdout, r.stdout + r.stderr


@pytest.fixture(scope="module")
def ema():
    import ema_attn

    ema_attn.lib()
    return ema_attn


ARGS = {
    "ema_causal_conv": dict(x=P, ldx=64, w=P, bias=P, starts=P, offsets=P, slots=P, batch=2, n_rows=5, max_rows=4,
                            channels=64, width=4, flags=1, state=P, n_slots=3, y=2 * P, ldy=64, dtype=1),
    "ema_ssm_scan": dict(x=P, ldx=128, dt=P, lddt=4, b=P, ldb=32, c=P, ldc=32, a=P, d=P, dt_bias=P, dt_min=0.0,
                         dt_max=INF, starts=P, offsets=P, slots=P, batch=2, n_rows=5, max_rows=4, heads=4, head_dim=32,
                         groups=2, d_state=16, flags=1, state=P, n_slots=3, y=2 * P, ldy=128, dtype=1, ws=P, bytes=1 << 30),
    "ema_gated_norm": dict(x=P, ldx=64, gate=P, ldg=64, w=P, eps=1e-6, n_rows=3, dim=64, group=16, flags=0, y=2 * P,
                           ldy=64, dtype=1),
    "ema_residual_norm": dict(branch=P, ldx=64, post_w=P, gate=P, ldg=64, scale=1.0, residual=2 * P, ldr=64, rdtype=4,
                              pre_w=P, eps=1e-6, n_rows=3, dim=64, flags=0, out=3 * P, ldo=64, dtype=1),
}


def call(ema, op, **over):
    a = dict(ARGS[op])
    assert not set(over) - set(a)
    a.update(over)
    return getattr(ema.lib(), op)(None, *a.values())


INVALID, SHAPE, CAPACITY, UNSUPPORTED = -1, -2, -3, -5
REFUSED = [
    ("ema_causal_conv", INVALID, [dict(x=0), dict(w=0), dict(y=0), dict(dtype=2), dict(flags=2), dict(x=P + 1), dict(y=P),
                                  dict(state=P + 1), dict(dtype=4, w=P + 2)]),
    ("ema_causal_conv", SHAPE, [dict(batch=0), dict(n_rows=-1), dict(max_rows=-1), dict(channels=0), dict(ldx=63),
                                dict(ldy=63), dict(starts=0), dict(n_slots=0)]),
    ("ema_causal_conv", UNSUPPORTED, [dict(width=1), dict(width=5), dict(batch=4097), dict(n_rows=(1 << 30) + 1),
                                      dict(channels=(1 << 21) + 1, ldx=1 << 22, ldy=1 << 22)]),
    ("ema_causal_conv", CAPACITY, [dict(slots=0, n_slots=1)]),
    ("ema_ssm_scan", INVALID, [dict(x=0), dict(dt=0), dict(b=0), dict(c=0), dict(a=0), dict(state=0), dict(y=0),
                               dict(dtype=0), dict(flags=2), dict(b=P + 4), dict(ldb=34), dict(ldc=34), dict(state=P + 8),
                               dict(a=P + 2), dict(dt=P + 1), dict(y=P), dict(ws=P + 8), dict(dt_min=1.0, dt_max=0.5),
                               dict(dt_min=NAN), dict(dt_max=NAN)]),
    ("ema_ssm_scan", SHAPE, [dict(ldx=127), dict(ldy=127), dict(lddt=3), dict(ldb=28), dict(ldc=28), dict(heads=0),
                             dict(head_dim=0), dict(groups=0), dict(groups=3), dict(d_state=0), dict(starts=0),
                             dict(batch=-1), dict(n_slots=-1)]),
    ("ema_ssm_scan", UNSUPPORTED, [dict(d_state=18, ldb=64, ldc=64), dict(d_state=260, ldb=1024, ldc=1024),
                                   dict(head_dim=4097, ldx=1 << 20, ldy=1 << 20), dict(batch=4097),
                                   dict(heads=65536, ldx=1 << 30, ldy=1 << 30, lddt=1 << 20),
                                   dict(batch=4096, slots=0, n_slots=4096, heads=512, groups=1, head_dim=128, ldx=1 << 16,
                                        ldy=1 << 16, lddt=512)]),
    ("ema_ssm_scan", CAPACITY, [dict(slots=0, n_slots=1)]),
    ("ema_gated_norm", INVALID, [dict(x=0), dict(y=0), dict(dtype=5), dict(flags=16), dict(eps=-1.0), dict(eps=NAN),
                                 dict(gate=P + 1), dict(y=P, ldy=72), dict(gate=3 * P, y=3 * P, ldy=72)]),
    ("ema_gated_norm", SHAPE, [dict(n_rows=-1), dict(dim=0), dict(group=0), dict(group=24), dict(ldx=63), dict(ldg=63),
                               dict(ldy=63)]),
    ("ema_gated_norm", UNSUPPORTED, [dict(dim=16392, group=16392, ldx=20000, ldg=20000, ldy=20000),
                                     dict(n_rows=1 << 30), dict(n_rows=1 << 22, dim=1024, group=1024, ldx=1024, ldg=1024, ldy=1024)]),
    ("ema_residual_norm", INVALID, [dict(branch=0), dict(residual=0), dict(out=0), dict(pre_w=0), dict(dtype=0),
                                    dict(rdtype=3), dict(dtype=4, rdtype=1), dict(flags=1), dict(eps=NAN),
                                    dict(residual=P), dict(out=2 * P), dict(out=P, ldo=72, gate=0), dict(gate=2 * P),
                                    dict(gate=3 * P), dict(residual=2 * P + 2), dict(branch=P + 1)]),
    ("ema_residual_norm", SHAPE, [dict(n_rows=-1), dict(dim=0), dict(ldx=63), dict(ldr=63), dict(ldo=63), dict(ldg=63)]),
    ("ema_residual_norm", UNSUPPORTED, [dict(dim=16385, ldx=20000, ldg=20000, ldr=20000, ldo=20000), dict(n_rows=1 << 22)]),
]


REFUSED += [
    ("ema_ssm_scan", INVALID, [dict(dt_min=-0.5), dict(dt_min=-INF)]),
    # a state of more than 2^30 values
    ("ema_ssm_scan", UNSUPPORTED, [dict(heads=4096, head_dim=4096, d_state=256, groups=1, ldx=1 << 24, ldy=1 << 24, lddt=4096,
                                        ldb=256, ldc=256)]),
]


@pytest.mark.parametrize("op,code,overs", REFUSED, ids=lambda v: str(v)[:24])
def test_refused_on_the_host(ema, op, code, overs):
    for over in overs:
        assert call(ema, op, **over) == code, (op, over, ema.last_error())
        assert op in ema.last_error()


def test_no_rows_is_no_work(ema):
    for op in ARGS:
        assert call(ema, op, n_rows=0) == ema.EMA_OK, ema.last_error()
    assert call(ema, "ema_causal_conv", n_rows=0, x=0, y=0) == ema.EMA_OK


def test_workspace_size(ema):
    size = ema.ssm_workspace_size
    assert size(1, 1, 1, 64, 64, 128, 8) == 0
    assert size(64, 64, 1, 64, 64, 128, 8) == 0
    long = size(1, 8192, 8192, 64, 64, 128, 8)
    assert 0 < long < 1 << 30
    assert size(1, 0, 0, 64, 64, 128, 8) == 0
    out = ctypes.c_uint64(7)
    for bad in [(0, 1, 1, 4, 32, 16, 2, 1), (1, -1, 1, 4, 32, 16, 2, 1), (1, 1, 1, 4, 32, 18, 2, 1),
                (1, 1, 1, 4, 32, 16, 3, 1), (1, 1, 1, 4, 32, 16, 2, 2)]:
        assert ema.lib().ema_ssm_workspace_size(*bad, ctypes.byref(out)) != ema.EMA_OK
    assert ema.lib().ema_ssm_workspace_size(1, 1, 1, 4, 32, 16, 2, 1, None) == ema.EMA_ERR_INVALID_ARG


def test_bindings_refuse_by_name(ema):
    torch = pytest.importorskip("torch")
    bf, f32 = torch.bfloat16, torch.float32
    z = lambda *s, d=bf: torch.zeros(*s, dtype=d)  # noqa: E731
    x, w = z(4, 16), z(16, 4)

    def refused(name, f, *a, **k):
        with pytest.raises(ema.EmaError) as e:
            f(*a, **k)
        assert name in str(e.value), str(e.value)

    conv = ema.causal_conv
    refused("weight", conv, x, z(8, 4), batch=1)
    refused("weight", conv, x, z(16, 4, d=f32), batch=1)
    refused("bias", conv, x, w, bias=z(8), batch=1)
    refused("state", conv, x, w, state=z(2, 4, 16), batch=1)
    refused("slots", conv, x, w, slots=torch.zeros(3, dtype=torch.int64))
    refused("slots", conv, x, w, slots=torch.zeros(3, dtype=torch.int32), offsets=torch.zeros(2, dtype=torch.int32))
    refused("x", conv, x.t(), z(4, 4), batch=1)
    refused("x must be", conv, x[0], w, batch=1)
    refused("weight", conv, x, None, batch=1)
    refused("dtype", conv, x.double(), w, batch=1)
    refused("out", conv, x, w, out=z(4, 8), batch=1)
    refused("GPU", conv, x, w, batch=1)
    a = dict(x=z(4, 2, 8), dt=z(4, 2), B=z(4, 1, 16), C=z(4, 1, 16), A=z(2, d=f32), state=z(1, 2, 8, 16, d=f32))
    for name, bad in [("dt", z(4, 3)), ("C", z(4, 1, 12)), ("C", z(4, 1, 16, d=f32)), ("A", z(2)), ("state", z(1, 2, 8, 16)),
                      ("state", z(1, 2, 8, 12, d=f32)), ("D", z(2)), ("dt_bias", z(3, d=f32)), ("B", None), ("state", None),
                      ("A", None), ("workspace", z(8)), ("out", z(4, 2, 9)), ("starts", torch.zeros(2, dtype=torch.int64))]:
        refused(name, ema.ssm_scan, **{**a, name: bad})
    refused("GPU", ema.ssm_scan, **a)
    refused("gate", ema.gated_norm, x, z(4, 8), z(16), 1e-6)
    refused("weight", ema.gated_norm, x, x, z(8), 1e-6)
    refused("residual", ema.residual_norm, x, z(4, 8), z(16), 1e-6)
    refused("residual", ema.residual_norm, x, None, z(16), 1e-6)
    refused("post_weight", ema.residual_norm, x, x.clone(), z(16), 1e-6, post_weight=z(8))
    refused("gate", ema.residual_norm, x, x.clone(), z(16), 1e-6, gate=z(8))
