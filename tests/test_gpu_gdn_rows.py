"""The Gated DeltaNet scan of pieces of a convolution's rows: the binding reads the values that its arguments hold,
not what lies behind their first element."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
from test_gpu_gdn import check_against_oracle  # noqa: E402
from test_gpu_mixer import BF, ema, rand  # noqa: E402,F401


@pytest.mark.parametrize("T", [1, 7, 70])
@pytest.mark.parametrize("space", [False, True])
def test_scan_of_a_convolutions_rows(ema, ora, T, space):
    Hk, Hv, Dk, Dv = 2, 4, 128, 128
    qkv, w = rand(1100, T, 2 * Hk * Dk + Hv * Dv, dtype=BF), rand(1101, 2 * Hk * Dk + Hv * Dv, 4, dtype=BF, scale=0.05)
    q, k, v = ema.causal_conv(qkv, w, batch=1).split([Hk * Dk, Hk * Dk, Hv * Dv], 1)
    q, k, v = q.view(1, T, Hk, Dk), k.view(1, T, Hk, Dk), v.view(1, T, Hv, Dv)
    gates = (torch.sigmoid(rand(1102, 1, Hv, T) + 3).transpose(1, 2), torch.sigmoid(rand(1103, 1, T, 2 * Hv))[:, :, ::2])
    start = rand(1104, 1, Hv, Dv, Dk, scale=0.3)
    ws = ema.gdn_workspace(1, T, Hk, Hv, Dk, Dv) if space else None
    state, packed = start.clone(), start.clone()
    y = ema.gdn_scan(q, k, v, *gates, state, workspace=ws)
    near = ema.gdn_scan(*(t.clone(memory_format=torch.contiguous_format) for t in (q, k, v, *gates)), packed, workspace=ws)
    torch.cuda.synchronize()
    assert torch.equal(y, near) and torch.equal(state, packed)
    host = [t.float().cpu().numpy() for t in (q, k, v, *gates, start)]
    check_against_oracle(ora, y, state, host, "bf16", f"{T} rows")


def test_scan_of_views_on_another_stream(ema):
    """The copies belong to the stream that is given."""
    T, Hk, Hv, D = 40, 2, 2, 64
    qkv = rand(1110, T, 3 * 2 * D, dtype=BF, scale=0.05)
    q, k, v = (t.view(1, T, 2, D) for t in qkv.split([2 * D] * 3, 1))
    g, beta = torch.sigmoid(rand(1111, 1, T, Hv)), torch.sigmoid(rand(1112, 1, T, Hv))
    want = torch.zeros(1, Hv, D, D, device="cuda")
    y = ema.gdn_scan(q, k, v, g, beta, want)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        state = torch.zeros(1, Hv, D, D, device="cuda")
        torch.cuda.synchronize()
        got = ema.gdn_scan(q, k, v, g, beta, state, stream=side)
        torch.cuda.synchronize()
        assert torch.equal(got, y) and torch.equal(state, want)
