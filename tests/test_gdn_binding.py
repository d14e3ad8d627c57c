"""The Python binding of the Gated DeltaNet scan refuses what the library, which takes bare pointers, would read wrongly."""
import pytest

torch = pytest.importorskip("torch")
import ema_attn as ema  # noqa: E402

BF, F32 = torch.bfloat16, torch.float32


def args(B=1, T=6, Hk=2, Hv=4, Dk=64, Dv=32):
    return dict(q=torch.zeros(B, T, Hk, Dk, dtype=BF), k=torch.zeros(B, T, Hk, Dk, dtype=BF), v=torch.zeros(B, T, Hv, Dv, dtype=BF),
                g=torch.zeros(B, T, Hv), beta=torch.zeros(B, T, Hv), state=torch.zeros(B, Hv, Dv, Dk))


@pytest.mark.parametrize("name,bad", [
    ("k", lambda: torch.zeros(1, 6, 2, 64)), ("k", lambda: torch.zeros(1, 6, 1, 64, dtype=BF)),
    ("v", lambda: torch.zeros(1, 5, 4, 32, dtype=BF)), ("v", lambda: torch.zeros(6, 4, 32, dtype=BF)),
    ("g", lambda: torch.zeros(1, 6, 4, dtype=BF)), ("g", lambda: torch.zeros(1, 4, 6)), ("beta", lambda: torch.zeros(1, 6, 8)),
    ("state", lambda: torch.zeros(1, 4, 64, 32).transpose(2, 3)), ("state", lambda: torch.zeros(1, 4, 32, 64, dtype=BF)),
    ("y", lambda: torch.zeros(1, 6, 4, 64, dtype=BF)[..., :32])])
def test_refused_by_name(name, bad):
    with pytest.raises(ema.EmaError) as e:
        ema.gdn_scan(**{**args(), name: bad()})
    assert f"{name} must be" in str(e.value) or (bad().dim() == 3 and "v [B,T,Hv,Dv]" in str(e.value))


def test_host_tensors_are_refused():
    with pytest.raises(ema.EmaError, match="GPU"):
        ema.gdn_scan(**args())
    with pytest.raises(ema.EmaError, match="workspace"):
        ema.gdn_scan(**args(), workspace=torch.zeros(64, dtype=torch.uint8)[::2])
