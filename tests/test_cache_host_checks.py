"""Host-side checks of the 8-bit cache entry points: status codes and Python errors without a GPU."""
import pytest
import torch

import gdn
from gdn import _lib, build


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def _append(lib, code=0, pages=4, P=16, max_pages=2, B=1, T=3, Hkv=2, D=128, len64=0, cu64=0, flags=0, **at):
    p = dict(k=256, v=256, kc=256, vc=256, ks=256, vs=256, table=256, lens=256, cu=256)
    p.update(at)
    return lib.gdn_cache_append(p["k"], p["v"], p["kc"], p["vc"], p["ks"], p["vs"], code, p["table"], p["lens"], len64, p["cu"],
                                cu64, pages, P, max_pages, B, T, Hkv, D, None, flags)


def _attend(lib, code=0, pages=4, P=16, max_pages=2, B=1, Q=1, Hq=4, Hkv=2, D=128, len64=0, ws=256, ws_bytes=1 << 30, flags=0, **at):
    p = dict(q=256, kc=256, vc=256, ks=256, vs=256, table=256, lens=256, out=256)
    p.update(at)
    return lib.gdn_cache_attend(p["q"], p["kc"], p["vc"], p["ks"], p["vs"], code, p["table"], p["lens"], len64, pages, P, max_pages,
                                B, Q, Hq, Hkv, D, 1.0, p["out"], ws, ws_bytes, None, flags)


@pytest.mark.parametrize("call", [_append, _attend])
def test_cache_status_codes(lib, call):
    assert call(lib, D=64) == 2 and call(lib, Hkv=0) == 2 and call(lib, Hkv=32768) == 2
    for kw in (dict(code=2), dict(P=8), dict(P=48), dict(P=256), dict(pages=-1), dict(max_pages=-1), dict(B=-1), dict(len64=2),
               dict(flags=1), dict(max_pages=1 << 28)):
        assert call(lib, **kw) == 4, kw
    for name in ("kc", "vc", "ks", "vs", "table", "lens"):
        assert call(lib, **{name: None}) == 1, name
    for kw in (dict(kc=264), dict(vc=264), dict(ks=258), dict(vs=258), dict(table=258), dict(lens=258), dict(lens=260, len64=1)):
        assert call(lib, **kw) == 3, kw
    assert call(lib, B=0) == 0


def test_append_status_codes(lib):
    assert _append(lib, T=-1) == 4 and _append(lib, cu64=2) == 4
    assert _append(lib, T=0) == 0 and _append(lib, pages=0) == 0 and _append(lib, max_pages=0) == 0
    for name in ("k", "v", "cu"):
        assert _append(lib, **{name: None}) == 1
    assert _append(lib, k=264) == 3 and _append(lib, v=264) == 3 and _append(lib, cu=258) == 3


def test_attend_status_codes(lib):
    assert _attend(lib, Hq=3) == 2 and _attend(lib, Hq=1) == 2
    assert _attend(lib, Q=-1) == 4 and _attend(lib, Q=1 << 30, B=1 << 10) == 4
    assert _attend(lib, Q=0) == 0
    assert _attend(lib, q=None) == 1 and _attend(lib, out=None) == 1
    assert _attend(lib, q=264) == 3 and _attend(lib, out=264) == 3
    assert _attend(lib, ws=None) == 5 and _attend(lib, ws=264) == 5 and _attend(lib, ws_bytes=1000) == 5
    assert lib.gdn_cache_attend_workspace_bytes() % 256 == 0


def test_python_refuses_cpu_tensors():
    q = torch.zeros(1, 1, 4, 128, dtype=torch.bfloat16)
    c, s = torch.zeros(2, 2, 16, 128, dtype=torch.int8), torch.zeros(2, 2)
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        gdn.cache_attend.run(q, c, c, s, s, i[None], i, None)
    with pytest.raises(ValueError, match="CUDA"):
        gdn.cache_append.kernel(q[0, :, :2], q[0, :, :2], c, c, s, s, i[None], i, torch.tensor([0, 1]))


@pytest.mark.parametrize("call", [_append, _attend])
@pytest.mark.parametrize("P", [16, 128])
def test_rows_of_the_table_hold_at_most_2_30_tokens(lib, call, P):
    """Above it, positions behind a sequence's end would not be ints."""
    empty = dict(T=0) if call is _append else dict(Q=0)
    assert call(lib, P=P, max_pages=(1 << 30) // P, **empty) == 0
    assert call(lib, P=P, max_pages=(1 << 30) // P + 1, **empty) == 4
    assert call(lib, P=P, max_pages=((1 << 31) - P) // P, **empty) == 4
