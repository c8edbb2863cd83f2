"""Host-side checks of the linear-attention entry points: status codes and Python errors without a GPU."""
import pytest
import torch

import gdn
from gdn import _lib, build


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def _decode(lib, B=1, H=4, HV=8, K=128, V=128, per_token=0, flags=0, **at):
    p = dict(q=256, k=256, v=256, state=256, decay=256, out=256, ns=256)
    p.update(at)
    return lib.gdn_linear_decode_fwd(p["q"], p["k"], p["v"], p["state"], p["decay"], per_token, 1.0, p["out"], p["ns"],
                                     B, H, HV, K, V, None, flags)


def _prefill(lib, N=1, T=64, H=4, HV=8, K=128, V=128, per_token=0, cu64=0, ws=256, ws_bytes=1 << 40, flags=0, **at):
    p = dict(q=256, k=256, v=256, state=256, decay=256, cu=256, out=256, ns=256)
    p.update(at)
    return lib.gdn_linear_prefill_fwd(p["q"], p["k"], p["v"], p["state"], p["decay"], per_token, p["cu"], cu64, N, T, 1.0,
                                      p["out"], p["ns"], ws, ws_bytes, H, HV, K, V, None, flags)


def test_decode_status_codes(lib):
    assert _decode(lib, H=3) == 2 and _decode(lib, K=64) == 2 and _decode(lib, HV=512, H=4) == 2
    assert _decode(lib, B=-1) == 4 and _decode(lib, per_token=2) == 4 and _decode(lib, flags=4) == 4
    assert _decode(lib, B=0, q=None) == 0
    assert _decode(lib, B=1 << 30) == 4  # more CTAs than a grid holds
    for name in ("q", "k", "v", "decay", "out", "ns"):
        assert _decode(lib, **{name: None}) == 1
    for name in ("q", "k", "v", "state", "out", "ns"):
        assert _decode(lib, **{name: 264}) == 3
    assert _decode(lib, decay=258) == 3


def test_prefill_status_codes(lib):
    assert _prefill(lib, H=3) == 2 and _prefill(lib, V=64) == 2
    assert _prefill(lib, N=-1) == 4 and _prefill(lib, T=-1) == 4 and _prefill(lib, cu64=2) == 4
    assert _prefill(lib, per_token=-1) == 4 and _prefill(lib, flags=8) == 4
    assert _prefill(lib, N=0) == 0
    for name in ("q", "k", "v", "decay", "cu", "out", "ns"):
        assert _prefill(lib, **{name: None}) == 1
    for name in ("q", "k", "v", "state", "out", "ns"):
        assert _prefill(lib, **{name: 264}) == 3
    assert _prefill(lib, cu=258) == 3 and _prefill(lib, cu=260, cu64=1) == 3
    assert _prefill(lib, ws=None) == 5 and _prefill(lib, ws=264) == 5 and _prefill(lib, T=8192, ws_bytes=4096) == 5


def test_prefill_workspace(lib):
    w = lib.gdn_linear_prefill_workspace_bytes
    assert w(1, 64, 4, 8, 128, 128) == 256  # one segment: the status word alone
    assert w(1, 8192, 4, 8, 128, 128) > w(1, 64, 4, 8, 128, 128)
    assert w(1, 64, 3, 8, 128, 128) == 0 and w(-1, 64, 4, 8, 128, 128) == 0
    # many short sequences need no state slots of their own
    assert w(20000, 60000, 4, 8, 128, 128) < 64 << 20
    assert w(64, 262144, 4, 8, 128, 128) < 1 << 30


def test_python_refuses_cpu_tensors():
    q, v = torch.zeros(4, 1, 4, 128, dtype=torch.bfloat16), torch.zeros(4, 1, 8, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        gdn.linear_decode.run(q, q, v, None, torch.zeros(8), None)
    with pytest.raises(ValueError, match="CUDA"):
        gdn.linear_prefill.run(q[:, 0], q[:, 0], v[:, 0], None, torch.zeros(8), torch.tensor([0, 4]), None)


def test_decay_shapes():
    from gdn._common import decay_rows
    cpu = torch.device("cpu")
    for bad in (torch.zeros(7), torch.zeros(5, 8), torch.zeros(6, 1, 7), torch.zeros(6, 2, 8)):
        with pytest.raises(ValueError):
            decay_rows(bad, 6, 8, cpu)
    with pytest.raises(TypeError):
        decay_rows(None, 6, 8, cpu)
    assert decay_rows(torch.zeros(8), 6, 8, cpu)[1] == 0
    assert decay_rows(torch.zeros(6, 8), 6, 8, cpu)[1] == 1
    assert decay_rows(torch.zeros(6, 1, 8), 6, 8, cpu)[1] == 1
