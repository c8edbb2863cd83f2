"""The 8-bit paged cache on the GPU: appending bit for bit, attention against 64 bits."""
import pytest
import torch

import gdn
from tests import cache_ref as ref

pytestmark = pytest.mark.gpu
SCALE = 128 ** -0.5


def _rows(T, Hkv, seed=0, spread=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((T, Hkv, 128), generator=g)
    if spread:  # rows of different sizes, so that scales grow inside a page
        x = x * torch.exp(torch.randn((T, 1, 1), generator=g))
    return x.to(torch.bfloat16)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Filled:
    """A cache filled in two calls: prompts, then a few more tokens for every sequence."""

    def __init__(self, lens, Hkv, P, code, seed=0, more=None, len_dtype=torch.int32):
        more = [min(n, 2) for n in lens] if more is None else more
        first = [n - m for n, m in zip(lens, more)]
        self.table, pages = ref.tables(lens, P, seed=seed)
        self.kc, self.vc, self.ks, self.vs = ref.empty_cache(pages, Hkv, P, code, seed=seed)
        self.lens, self.code = lens, code
        self.seq = torch.tensor(lens, dtype=len_dtype, device="cuda")
        for part, total in ((first, first), (more, lens)):
            cu = [0]
            for n in part:
                cu.append(cu[-1] + n)
            k, v = _rows(cu[-1], Hkv, seed + 1).cuda(), _rows(cu[-1], Hkv, seed + 2).cuda()
            want = [ref.append(x, c, s, self.table, total, cu, code) for x, c, s in ((k, self.kc, self.ks), (v, self.vc, self.vs))]
            gdn.cache_append.kernel(k, v, self.kc, self.vc, self.ks, self.vs, self.table,
                                    torch.tensor(total, dtype=len_dtype, device="cuda"), _i32(cu))
            for (raw, sc), c, s in zip(want, (self.kc, self.vc), (self.ks, self.vs)):
                assert torch.equal(c.view(torch.uint8).cpu(), torch.from_numpy(raw))
                assert torch.equal(s.cpu().nan_to_num(-1), torch.from_numpy(sc).nan_to_num(-1))

    def args(self):
        return self.kc, self.vc, self.ks, self.vs, self.table

    def q(self, Q, Hq, seed=5):
        g = torch.Generator().manual_seed(seed)
        return (torch.randn((len(self.lens), Q, Hq, 128), generator=g) * 2).to(torch.bfloat16).cuda()

    def check(self, q, out, scale=SCALE, rows=slice(None)):
        want, tol = ref.attend(q, *self.args(), self.lens, scale)
        e = (out.double() - want).abs()
        assert (e <= tol)[rows].all(), f"off by {(e / tol)[rows].max().item():.2f} times the bound"


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("P", [16, 32, 64, 128])
@pytest.mark.parametrize("lens", [[1], [15, 16, 17], [0, 300, 1, 64, 0, 129], [33] * 40])
def test_append_and_decode(code, P, lens):
    f = Filled(lens, 2, P, code, seed=P)
    q = f.q(1, 8)
    out = gdn.cache_attend.run(q, *f.args(), f.seq, SCALE)
    f.check(q, out)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("Q", [1, 2, 5, 16])
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (8, 8), (12, 1), (32, 2), (15, 3)])
def test_head_layouts_and_several_tokens(code, Q, Hq, Hkv):
    f = Filled([70, 3, 500], Hkv, 32, code, seed=Q)
    q = f.q(Q, Hq)
    f.check(q, gdn.cache_attend.run(q, *f.args(), f.seq, SCALE))


@pytest.mark.parametrize("lens", [[20000], [9000, 1, 40], [5000, 0, 2500, 2500]])
def test_long_caches_are_split_and_joined(lens):
    f = Filled(lens, 1, 64, "e4m3", more=[0] * len(lens), len_dtype=torch.int64)
    q = f.q(3, 8)
    ws = torch.empty(gdn.cache_attend.workspace_bytes(), dtype=torch.uint8, device="cuda").fill_(255)
    out = torch.empty_like(q)
    gdn.cache_attend.kernel(q, *f.args(), f.seq, SCALE, out, workspace=ws)
    f.check(q, out)
    assert gdn.cache_attend.read_status(ws) == 0
    again = gdn.cache_attend.run(q, *f.args(), f.seq, SCALE)
    assert torch.equal(out, again)


def test_many_sequences():
    f = Filled([(37 * i) % 50 for i in range(700)], 1, 16, "int8", more=[0] * 700)
    q = f.q(1, 4)
    f.check(q, gdn.cache_attend.run(q, *f.args(), f.seq, SCALE))


def test_decode_steps_grow_the_cache():
    """Token by token from nothing, scales growing inside every page, against one reference that follows along."""
    lens, Hkv, P = [0, 13, 31], 2, 16
    table, pages = ref.tables([n + 40 for n in lens], P)
    kc, vc, ks, vs = ref.empty_cache(pages, Hkv, P, "int8")
    start = _rows(sum(lens), Hkv, 3).cuda()
    gdn.cache_append.kernel(start, start, kc, vc, ks, vs, table, _i32(lens), _i32([0, 0, 13, 44]))
    for step in range(40):
        lens = [n + 1 for n in lens]
        x = (_rows(3, Hkv, 100 + step) * (1 + 0.1 * step)).to(torch.bfloat16).cuda()
        want = ref.append(x, kc, ks, table, lens, [0, 1, 2, 3], "int8")
        gdn.cache_append.kernel(x, x, kc, vc, ks, vs, table, _i32(lens), _i32([0, 1, 2, 3]))
        assert torch.equal(kc.view(torch.uint8).cpu(), torch.from_numpy(want[0]))
        q = torch.randn((3, 1, 8, 128), device="cuda").to(torch.bfloat16)
        out = gdn.cache_attend.run(q, kc, vc, ks, vs, table, _i32(lens), None)
        o, tol = ref.attend(q, kc, vc, ks, vs, table, lens, SCALE)
        assert ((out.double() - o).abs() <= tol).all()


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_rows_that_see_nothing(code):
    f = Filled([0, 2, 1, 40], 2, 16, code)
    q = f.q(4, 4)
    out = gdn.cache_attend.run(q, *f.args(), f.seq, SCALE)
    assert not out[0].any() and not out[1, :2].any() and not out[2, :3].any()
    f.check(q, out)


def test_zero_and_uneven_scales():
    """Pages of nothing but zeros (scale 0) between pages of very different value scales."""
    lens, P = [200, 64], 16
    table, pages = ref.tables(lens, P)
    kc, vc, ks, vs = ref.empty_cache(pages, 1, P, "int8")
    k, v = _rows(264, 1, 1), _rows(264, 1, 2, spread=False).float()
    for i in range(264):
        v[i] *= [0.0, 1e-20, 1e4, 1.0, 1e-3][(i // 16) % 5]
    v = v.to(torch.bfloat16)
    k[16:32] = 0
    gdn.cache_append.kernel(k.cuda(), v.cuda(), kc, vc, ks, vs, table, _i32(lens), _i32([0, 200, 264]))
    q = torch.randn((2, 1, 4, 128), device="cuda").to(torch.bfloat16)
    out = gdn.cache_attend.run(q, kc, vc, ks, vs, table, _i32(lens), SCALE)
    o, tol = ref.attend(q, kc, vc, ks, vs, table, lens, SCALE)
    assert ((out.double() - o).abs() <= tol).all()


@pytest.mark.parametrize("factor", [1e-30, 1e-4, 1e4, 1e30])
def test_sizes_of_q(factor):
    """q far outside fp16's range in either direction; the scale brings the scores back."""
    f = Filled([100], 1, 32, "e4m3")
    q = (f.q(2, 4).float() * factor).to(torch.bfloat16)
    f.check(q, gdn.cache_attend.run(q, *f.args(), f.seq, SCALE / factor), scale=SCALE / factor)


def test_nan_in_q_reaches_its_row_only():
    f = Filled([100, 20], 1, 32, "e4m3")
    q = f.q(1, 4)
    want = gdn.cache_attend.run(q, *f.args(), f.seq, SCALE)
    q[0, 0, 2, 7] = float("nan")
    out = gdn.cache_attend.run(q, *f.args(), f.seq, SCALE)
    assert out[0, 0, 2].isnan().all()
    keep = [0, 1, 3]
    assert torch.equal(out[0, 0, keep], want[0, 0, keep]) and torch.equal(out[1], want[1])


def test_append_of_infinities_and_nan():
    for code in ("int8", "e4m3"):
        table, pages = ref.tables([20], 16)
        kc, vc, ks, vs = ref.empty_cache(pages, 1, 16, code)
        x = _rows(20, 1)
        x[3, 0, 5], x[4, 0, 6], x[7, 0, 0] = float("inf"), float("-inf"), float("nan")
        x[18] = 0
        x[17, 0, 1] = float("nan")
        want = ref.append(x, kc, ks, table, [20], [0, 20], code)
        gdn.cache_append.kernel(x.cuda(), x.cuda(), kc, vc, ks, vs, table, _i32([20]), _i32([0, 20]))
        got, exp = kc.view(torch.uint8).cpu(), torch.from_numpy(want[0])
        if code == "e4m3":  # a NaN has two codes
            got, exp = (torch.where((t & 0x7F) == 0x7F, torch.full_like(t, 0x7F), t) for t in (got, exp))
        assert torch.equal(got, exp)
        assert torch.equal(ks.cpu().nan_to_num(-1), torch.from_numpy(want[1]).nan_to_num(-1))


def test_append_of_zeros_and_tiny_values():
    for code in ("int8", "e4m3"):
        table, pages = ref.tables([40], 16)
        kc, vc, ks, vs = ref.empty_cache(pages, 2, 16, code)
        x = torch.zeros((40, 2, 128), dtype=torch.bfloat16)
        x[20:] = (_rows(20, 2).float() * 1e-38).to(torch.bfloat16)
        want = ref.append(x, kc, ks, table, [40], [0, 40], code)
        gdn.cache_append.kernel(x.cuda(), x.cuda(), kc, vc, ks, vs, table, _i32([40]), _i32([0, 40]))
        assert torch.equal(kc.view(torch.uint8).cpu(), torch.from_numpy(want[0]))
        assert torch.equal(ks.cpu().nan_to_num(-1), torch.from_numpy(want[1]).nan_to_num(-1))


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("size", [2.0 ** -100, 2.0 ** -62, 2.0 ** -55, 1.0, 2.0 ** 64, 2.0 ** 120])
def test_codes_are_those_of_the_quotients(code, size):
    """Values at and beside the halves between codes, zeros of both signs, over the range of fp32's scales."""
    g = torch.Generator().manual_seed(3)
    T, m = 48, 127 if code == "int8" else 448
    x = torch.randn((T, 1, 128), generator=g)
    top = x.abs().amax()
    x[:, :, 1::4] = top / 2 ** torch.randint(0, 14, (T, 1, 32), generator=g)
    x[:, :, 2::4] = top * (torch.randint(-m, m, (T, 1, 32), generator=g) + 0.5) / m
    x[::3, :, 3] = 0.0
    x[1::3, :, 3] = -0.0
    x = (x * size).to(torch.bfloat16)
    table, pages = ref.tables([T], 16)
    kc, vc, ks, vs = ref.empty_cache(pages, 1, 16, code)
    for n, part in ((7, x[:7]), (10, x[7:10]), (T, x[10:])):  # the last part grows a page's scale
        d = (part * (1.0 if n == T else 0.25)).cuda()
        cu = [0, part.shape[0]]
        want = [ref.append(y, c, s, table, [n], cu, code) for y, c, s in ((d, kc, ks), (-d, vc, vs))]
        gdn.cache_append.kernel(d, -d, kc, vc, ks, vs, table, _i32([n]), _i32(cu))
        for (raw, sc), c, s in zip(want, (kc, vc), (ks, vs)):
            assert torch.equal(s.cpu().nan_to_num(-1), torch.from_numpy(sc).nan_to_num(-1))
            assert torch.equal(c.view(torch.uint8).cpu(), torch.from_numpy(raw))


@pytest.mark.parametrize("lens", [[1] * 2500, [40, 0, 200] * 30, [33] * 40])
def test_append_to_many_sequences(lens):
    """Searches of several rounds; one warp a page, whose rows need several turns, and a warp for each 16 rows."""
    f = Filled(lens, 3, 64, "e4m3", more=[0] * len(lens))
    q = f.q(1, 3)
    f.check(q, gdn.cache_attend.run(q, *f.args(), f.seq, SCALE))


def test_padded_rows_and_bad_pages_drop_their_rows():
    """seq_lens 0 with a row given, a table too short, pages outside the cache: dropped, the rest is as ever."""
    table, pages = ref.tables([40, 40, 40, 40], 16)
    table[2, 1] = pages
    table[3, 0] = -1
    table = table[:, :2].contiguous()
    kc, vc, ks, vs = ref.empty_cache(pages, 2, 16, "int8")
    cu, lens = [0, 40, 41, 81, 121], [40, 0, 40, 40]
    x = _rows(121, 2)
    want = [ref.append(x, c, s, table, lens, cu, "int8") for c, s in ((kc, ks), (vc, vs))]
    gdn.cache_append.kernel(x.cuda(), x.cuda(), kc, vc, ks, vs, table, _i32(lens), _i32(cu))
    for (raw, sc), c, s in zip(want, (kc, vc), (ks, vs)):
        assert torch.equal(c.view(torch.uint8).cpu(), torch.from_numpy(raw))
        assert torch.equal(s.cpu().nan_to_num(-1), torch.from_numpy(sc).nan_to_num(-1))


def test_attend_reports_bad_pages_and_lengths():
    f = Filled([60, 60, 60], 1, 16, "e4m3")
    q = f.q(1, 4)
    want = gdn.cache_attend.run(q, *f.args(), f.seq, SCALE)
    ws = torch.empty(gdn.cache_attend.workspace_bytes(), dtype=torch.uint8, device="cuda")
    out = torch.empty_like(q)
    bad = f.table.clone()
    bad[1, 2] = -5
    gdn.cache_attend.kernel(q, f.kc, f.vc, f.ks, f.vs, bad, f.seq, SCALE, out, workspace=ws)
    assert gdn.cache_attend.read_status(ws) == 6
    assert torch.equal(out[0], want[0]) and torch.equal(out[2], want[2]) and torch.isfinite(out).all()
    gdn.cache_attend.kernel(q, *f.args(), _i32([60, 60, 1000]), SCALE, out, workspace=ws)
    assert gdn.cache_attend.read_status(ws) == 5
    assert torch.equal(out[:2], want[:2])
    gdn.cache_attend.kernel(q, *f.args(), f.seq, SCALE, out, workspace=ws)
    assert gdn.cache_attend.read_status(ws) == 0 and torch.equal(out, want)


def test_cache_beyond_32_bit_offsets():
    """A cache of more than 2^32 bytes, the sequence in its last pages."""
    pages, P = 300000, 128
    kc = torch.empty((pages, 1, P, 128), dtype=torch.int8, device="cuda")
    vc = torch.empty_like(kc)
    ks, vs = (torch.zeros((pages, 1), device="cuda") for _ in range(2))
    table = torch.tensor([[pages - 1, pages - 3, pages - 2]], dtype=torch.int32, device="cuda")
    k, v = _rows(300, 1, 1).cuda(), _rows(300, 1, 2).cuda()
    gdn.cache_append.kernel(k, v, kc, vc, ks, vs, table, _i32([300]), _i32([0, 300]))
    small = table[0].long()
    args = [x[small].contiguous() for x in (kc, vc, ks, vs)]
    t2 = _i32([[0, 1, 2]])
    want = ref.append(k, args[0], torch.zeros((3, 1)), t2, [300], [0, 300], "int8")
    n = 300 - 256
    assert torch.equal(args[0].view(torch.uint8).cpu()[:2], torch.from_numpy(want[0])[:2])
    assert torch.equal(args[0].view(torch.uint8).cpu()[2, :, :n], torch.from_numpy(want[0])[2, :, :n])
    q = torch.randn((1, 1, 4, 128), device="cuda").to(torch.bfloat16)
    a = gdn.cache_attend.run(q, kc, vc, ks, vs, table, _i32([300]), SCALE)
    b = gdn.cache_attend.run(q, *args, t2, _i32([300]), SCALE)
    assert torch.equal(a, b)


def test_captured_and_replayed_with_linear_layers():
    """One decode step of a stack, a linear-attention layer and a cache layer, captured once and replayed as the
    sequences grow; an eager run on copies of the state gives the same bits."""
    B, Hkv, Hq, P = 3, 2, 8, 16
    lens0 = [5, 16, 30]
    table, pages = ref.tables([n + 10 for n in lens0], P)
    g = torch.Generator().manual_seed(0)

    def fresh():
        kc, vc, ks, vs = ref.empty_cache(pages, Hkv, P, "e4m3")
        x = _rows(sum(lens0), Hkv, 1).cuda()
        gdn.cache_append.kernel(x, x, kc, vc, ks, vs, table, _i32(lens0), _i32([0, 5, 21, 51]))
        return dict(kc=kc, vc=vc, ks=ks, vs=vs, lens=_i32(lens0), cu=_i32([0, 1, 2, 3]),
                    state=torch.zeros((B, 8, 128, 128), device="cuda"), a=-0.1 * torch.ones(8, device="cuda"),
                    q=torch.zeros((B, 1, Hq, 128), dtype=torch.bfloat16, device="cuda"),
                    lo=torch.zeros((B, 1, 8, 128), dtype=torch.bfloat16, device="cuda"),
                    out=torch.zeros((B, 1, Hq, 128), dtype=torch.bfloat16, device="cuda"),
                    ws=torch.empty(gdn.cache_attend.workspace_bytes(), dtype=torch.uint8, device="cuda"))

    def step(s):
        s["lens"] += 1
        gdn.linear_decode.kernel(s["q"][:, :, :4], s["q"][:, :, 4:], s["q"], s["state"], s["a"], SCALE, s["lo"], s["state"])
        kv = s["lo"][:, 0, :Hkv]
        gdn.cache_append.kernel(kv, s["q"][:, 0, :Hkv], s["kc"], s["vc"], s["ks"], s["vs"], table, s["lens"], s["cu"])
        gdn.cache_attend.kernel(s["q"], s["kc"], s["vc"], s["ks"], s["vs"], table, s["lens"], SCALE, s["out"], workspace=s["ws"])

    warm = fresh()
    step(warm)
    torch.cuda.synchronize()
    a, b = fresh(), fresh()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(a)
    for _ in range(8):
        x = torch.randn((B, 1, Hq, 128), generator=g).to(torch.bfloat16)
        a["q"].copy_(x)
        b["q"].copy_(x)
        graph.replay()
        step(b)
        assert torch.equal(a["out"], b["out"]) and torch.equal(a["state"], b["state"])
        assert torch.equal(a["kc"].view(torch.uint8), b["kc"].view(torch.uint8))
        want, tol = ref.attend(b["q"], b["kc"], b["vc"], b["ks"], b["vs"], table, b["lens"].tolist(), SCALE)
        assert ((b["out"].double() - want).abs() <= tol).all()


def test_two_streams_with_workspaces_of_their_own():
    f = Filled([3000, 2000], 2, 64, "int8", more=[0, 0])
    qs = [f.q(1, 16, seed=s) for s in (1, 2)]
    want = [gdn.cache_attend.run(q, *f.args(), f.seq, SCALE) for q in qs]
    outs = [torch.empty_like(q) for q in qs]
    ws = [torch.empty(gdn.cache_attend.workspace_bytes(), dtype=torch.uint8, device="cuda") for _ in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, q, o, w in zip(streams, qs, outs, ws):
            with torch.cuda.stream(s):
                gdn.cache_attend.kernel(q, *f.args(), f.seq, SCALE, o, workspace=w)
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))


def test_nothing_to_do():
    f = Filled([20], 1, 16, "int8")
    q = f.q(1, 2)
    assert gdn.cache_attend.run(q[:, :0], *f.args(), f.seq, SCALE).numel() == 0
    assert gdn.cache_attend.run(q[:0], *f.args()[:4], f.table[:0], f.seq[:0], SCALE).numel() == 0
    before = f.kc.clone()
    x = torch.empty((0, 1, 128), dtype=torch.bfloat16, device="cuda")
    gdn.cache_append.kernel(x, x, *f.args()[:4], f.table, f.seq, _i32([0, 0]))
    assert torch.equal(before, f.kc)
    empty = torch.empty((0, 1, 16, 128), dtype=torch.int8, device="cuda")
    es = torch.empty((0, 1), device="cuda")
    out = gdn.cache_attend.run(q, empty, empty, es, es, f.table, f.seq, SCALE)
    assert not out.any()


def test_refusals():
    f = Filled([20], 2, 16, "int8")
    q = f.q(1, 4)
    A = gdn.cache_attend.run
    with pytest.raises(ValueError, match="multiple"):
        A(q[:, :, :3], *f.args(), f.seq, SCALE)
    with pytest.raises(ValueError, match="k_cache"):
        A(q, f.kc.to(torch.uint8), f.vc, f.ks, f.vs, f.table, f.seq, SCALE)
    with pytest.raises(ValueError, match="v_cache"):
        A(q, f.kc, f.vc[..., ::2], f.ks, f.vs, f.table, f.seq, SCALE)
    with pytest.raises(ValueError, match="same shape"):
        A(q, f.kc, f.vc[:1], f.ks, f.vs, f.table, f.seq, SCALE)
    with pytest.raises(ValueError, match="page size"):
        A(q, *(x[:, :, :8].contiguous() for x in (f.kc, f.vc)), f.ks, f.vs, f.table, f.seq, SCALE)
    with pytest.raises(ValueError, match="k_scale"):
        A(q, f.kc, f.vc, f.ks.double(), f.vs, f.table, f.seq, SCALE)
    with pytest.raises(ValueError, match="block_table"):
        A(q, *f.args()[:4], f.table[0], f.seq, SCALE)
    with pytest.raises(ValueError, match="seq_lens"):
        A(q, *f.args(), f.seq.float(), SCALE)
    with pytest.raises(ValueError, match="output"):
        gdn.cache_attend.kernel(q, *f.args(), f.seq, SCALE, q.float())
    with pytest.raises(ValueError, match="workspace"):
        gdn.cache_attend.kernel(q, *f.args(), f.seq, SCALE, torch.empty_like(q), workspace=q)
    with pytest.raises(ValueError, match="k and v"):
        gdn.cache_append.kernel(q[0], q[0], *f.args()[:4], f.table, f.seq, _i32([0, 1]))


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_append_of_infinities_and_nan_among_zeros(code):
    """The page's scale is 0 then; the codes are those of any other page, and stay when a later token brings a scale."""
    table, pages = ref.tables([10], 16)
    kc, vc, ks, vs = ref.empty_cache(pages, 1, 16, code)
    x = torch.zeros((6, 1, 128), dtype=torch.bfloat16)
    x[1, 0, 5], x[2, 0, 6], x[4, 0, 9], x[4, 0, 10] = float("inf"), float("-inf"), float("nan"), -0.0
    big, nan = (127, 0) if code == "int8" else (0x7E, 0x7F)
    minus = 129 if code == "int8" else 0xFE
    gdn.cache_append.kernel(x.cuda(), -x.cuda(), kc, vc, ks, vs, table, _i32([6]), _i32([0, 6]))
    page = table[0, 0].item()
    for c, s, inf, ninf in ((kc, ks, big, minus), (vc, vs, minus, big)):
        raw = c.view(torch.uint8)[page, 0, :6].cpu()
        assert s[page, 0] == 0
        assert raw[1, 5] == inf and raw[2, 6] == ninf
        assert (raw[4, 9] & (0x7F if code == "e4m3" else 0xFF)) == nan
        assert (raw.to(torch.int32) & 0x7F != 0).sum() == (3 if code == "e4m3" else 2)
    y = torch.ones((1, 1, 128), dtype=torch.bfloat16).cuda()
    gdn.cache_append.kernel(y, y, kc, vc, ks, vs, table, _i32([7]), _i32([0, 1]))
    raw = kc.view(torch.uint8)[page, 0, :7].cpu().to(torch.int32) & 0x7F
    assert ks[page, 0] > 0 and (raw[6] == big).all()
    assert (raw[4, 9] == 0x7F) if code == "e4m3" else raw[4, 9] == 0
    raw[4, 9] = 0
    assert not raw[:6].any()  # an infinity kept no size: 0 times its code


class Poked(Filled):
    """A filled cache some of whose codes and value scales are then overwritten; `rows` that see none of them keep their values."""

    def poke(self, b, token, head, dim, raw):
        P = self.vc.shape[2]
        self.vc.view(torch.uint8)[self.table[b, token // P].item(), head, token % P, dim] = raw

    def check_apart(self, q, clean, tol, dirty):
        """NaN (or infinite) exactly where `dirty` is, elsewhere as before the pokes."""
        out = gdn.cache_attend.run(q, *self.args(), self.seq, SCALE).double()
        hit = ~torch.isfinite(dirty)
        assert torch.equal(~torch.isfinite(out), hit)
        assert hit.any() and (((out - clean).abs() <= tol) | hit).all()


@pytest.mark.parametrize("Q,Hq,Hkv", [(2, 2, 2), (4, 8, 2), (3, 5, 1), (16, 8, 1), (33, 2, 1)])
@pytest.mark.parametrize("P", [16, 64])
def test_nan_in_v_reaches_only_rows_that_see_it(Q, Hq, Hkv, P):
    """e4m3 has a code for NaN: a later token's must not reach earlier rows, nor one that sees no token at all."""
    lens = [Q + 38, 3, 1, 500, 2, Q + 9]
    f = Poked(lens, Hkv, P, "e4m3", seed=Q, more=[0] * len(lens))
    q = f.q(Q, Hq)
    clean, tol = ref.attend(q, *f.args(), f.lens, SCALE)
    for b, n in enumerate(lens[:-1]):  # the last sequence stays clean
        f.poke(b, n - 1, Hkv - 1, 5, 0x7F)
        if n > 2:
            f.poke(b, n - 2, 0, 77, 0xFF)
            f.poke(b, n - 2, 0, slice(96, 128), 0x7F)
    f.poke(3, 100, Hkv - 1, 127, 0x7F)
    f.check_apart(q, clean, tol, ref.attend(q, *f.args(), f.lens, SCALE)[0])


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("Q", [2, 4, 20])
def test_value_scale_that_is_not_finite_reaches_only_rows_that_see_its_page(code, bad, Q):
    lens = [33, 65, 17]  # the last token begins a page
    f = Poked(lens, 1, 16, code, more=[0] * 3)
    f.vc.view(torch.uint8)[f.table[0, 2].item(), :, 0] = 0x11
    q = f.q(Q, 3)
    clean, tol = ref.attend(q, *f.args(), f.lens, SCALE)
    f.vs[f.table[0, 2].item()] = bad
    f.check_apart(q, clean, tol, ref.attend(q, *f.args(), f.lens, SCALE)[0])


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("ratio", [2.0 ** -100, 2.0 ** -20, 2.0 ** 12, 2.0 ** 17, 2.0 ** 30, 2.0 ** 45])
@pytest.mark.parametrize("Q,page", [(1, 0), (1, 150), (3, 7), (8, 255)])
def test_a_page_of_other_size_and_little_weight(code, ratio, Q, page):
    """Values `ratio` times as large in one page, whose scores are 2^-60 below the others': it must not cost the others
    their bits.  The bound is cache_ref's, but weights below fp16's normal range are measured by the row's largest
    weight times value scale, 2^-25 of it each, instead of the largest value in the cache."""
    n, P, Hq = 4096, 16, 4
    table, pages = ref.tables([n], P)
    kc, vc, ks, vs = ref.empty_cache(pages, 1, P, code)
    g = torch.Generator().manual_seed(7)
    k, v = (torch.randn((n, 1, 128), generator=g) for _ in range(2))
    q = (torch.randn((1, Q, Hq, 128), generator=g) * 0.1 + 1).to(torch.bfloat16).cuda()
    at = slice(page * P, (page + 1) * P)
    k[at] = k[at] * 0.1 - 60 * 0.69315 / SCALE / 128
    v[at] *= ratio
    gdn.cache_append.kernel(k.to(torch.bfloat16).cuda(), v.to(torch.bfloat16).cuda(), kc, vc, ks, vs, table, _i32([n]), _i32([0, n]))
    out = gdn.cache_attend.run(q, kc, vc, ks, vs, table, _i32([n]), SCALE).double()
    idx = table[0].long()
    K, V = ((c.view(torch.uint8)[idx, 0].view(c.dtype).double() * s[idx, 0].double()[:, None, None]).reshape(-1, 128) for c, s in ((kc, ks), (vc, vs)))
    size = vs[idx, 0].double().repeat_interleave(P) * (127 if code == "int8" else 448)
    for i in range(Q):
        m = n - Q + 1 + i
        qq = q[0, i].double()
        s = SCALE * (qq @ K[:m].T)
        d = SCALE * (2.0 ** -17 * (qq.abs() @ K[:m].abs().T) + 2.0 ** -24 * qq.abs().amax(-1, keepdim=True) * K[:m].abs().sum(-1)) + 2.0 ** -21 * s.abs()
        w = torch.softmax(s, -1)
        o = w @ V[:m]
        tol = 2.0 ** -8 * o.abs() + (2.0 ** -10 + 2 * d.amax(-1, keepdim=True)) * (w @ V[:m].abs()) + m * 2.0 ** -25 * (w * size[:m]).amax(-1, keepdim=True)
        e = (out[0, i] - o).abs()
        assert (e <= tol).all(), f"row {i} off by {(e / tol).max().item():.2f} times its bound"


def test_the_gravest_status_of_a_block_is_kept():
    """A bad page, then a sequence longer than its row of the table, wherever the two fall among the blocks."""
    f = Filled([20] * 700, 1, 16, "int8", more=[0] * 700)
    q = f.q(1, 2)
    ws = torch.empty(gdn.cache_attend.workspace_bytes(), dtype=torch.uint8, device="cuda")
    out = torch.empty_like(q)
    for b in range(300, 306):
        table, seq = f.table.clone(), f.seq.clone()
        table[b, 0] = -1
        seq[b + 1] = 1000
        gdn.cache_attend.kernel(q, *f.args()[:4], table, seq, SCALE, out, workspace=ws)
        assert gdn.cache_attend.read_status(ws) == 6
