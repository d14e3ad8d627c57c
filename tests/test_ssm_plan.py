"""The state space scan's plan without a GPU: the places of its workspace (tests/cpp/test_ssm_plan.cpp) and the sizes
that are told for it."""
import os
import subprocess

import pytest

CPP = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp")


def test_integer_parts():
    subprocess.run(["make", "-s", "-C", CPP, "test_ssm_plan"], check=True)
    r = subprocess.run([os.path.join(CPP, "test_ssm_plan")], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "checks passed" in r.stdout, r.stdout + r.stderr


@pytest.fixture(scope="module")
def size():
    import ema_attn

    ema_attn.lib()
    return ema_attn.ssm_workspace_size


def test_sequences_of_one_piece_take_no_state(size):
    """63 users' tokens beside a prompt: at most twice what the prompt needs alone."""
    alone = size(1, 8192, 8192, 64, 64, 128, 8)
    assert alone <= size(64, 8192 + 63, 8192, 64, 64, 128, 8) <= 2 * alone


def test_a_size_holds_every_smaller_call(size):
    """A server sizes its workspace once: many long prompts, of which none is cut, and one alone, which is."""
    assert size(8, 65536, 8192, 64, 64, 128, 8) >= size(1, 8192, 8192, 64, 64, 128, 8) > 0
    assert size(32, 32, 1, 64, 64, 128, 8) == 0 and size(512, 512, 1, 2, 64, 128, 1) == 0


def test_limits_that_the_header_tells():
    """The last number of rows that passes a limit is refused for what comes after it, the first beyond it for it."""
    import ema_attn as ema
    from test_mixer import INVALID, UNSUPPORTED, call

    ema.lib()
    wide = dict(dim=64, ldx=64, ldr=64, ldo=64, ldg=64)
    assert call(ema, "ema_residual_norm", n_rows=(1 << 22) - 1, branch=0, **wide) == INVALID
    assert call(ema, "ema_residual_norm", n_rows=1 << 22, branch=0, **wide) == UNSUPPORTED
    assert call(ema, "ema_gated_norm", n_rows=1 << 24, dim=64, group=16) == UNSUPPORTED
    assert call(ema, "ema_gated_norm", n_rows=1 << 21, dim=2048, group=1024, ldx=2048, ldg=2048, ldy=2048) == UNSUPPORTED
    # (groups of 512 values and fewer have the larger limit)
    assert call(ema, "ema_gated_norm", n_rows=1 << 22, dim=512, group=512, ldx=512, ldg=512, ldy=512, x=0) == INVALID
    assert call(ema, "ema_causal_conv", channels=1 << 21, ldx=1 << 22, ldy=1 << 22, y=1) == INVALID
    assert call(ema, "ema_causal_conv", channels=(1 << 21) + 1, ldx=1 << 22, ldy=1 << 22) == UNSUPPORTED
