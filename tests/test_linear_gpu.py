"""Linear attention with a decay for each head on the GPU against the token recurrence in 64 bits."""
import pytest
import torch

import gdn
from gdn import _lib
from tests import linear_ref as ref

pytestmark = pytest.mark.gpu
SCALE = 128 ** -0.5


def _cu(cu, dtype=torch.int32):
    return torch.tensor(cu, dtype=dtype, device="cuda")


def _run(x, cu_dtype=torch.int32):
    q, k, v, st, a, cu = x
    return gdn.linear_prefill.run(q, k, v, st, a, _cu(cu, cu_dtype), SCALE)


@pytest.mark.parametrize("B", [1, 2, 17, 64])
@pytest.mark.parametrize("H,HV", [(4, 8), (1, 1), (16, 32), (3, 9)])
@pytest.mark.parametrize("per_token", [False, True])
def test_decode(B, H, HV, per_token):
    q, k, v, st, a, cu = ref.inputs([1] * B, H, HV, seed=B, per_token=per_token)
    out, ns = gdn.linear_decode.run(q[:, None], k[:, None], v[:, None], st, a if not per_token else a[:, None], SCALE)
    assert out.shape == (B, 1, HV, 128) and out.dtype == torch.bfloat16
    ref.check(out[:, 0], ns, ref.reference(q, k, v, st, a, cu, SCALE), chunked=False)


def test_decode_without_state_and_in_place():
    q, k, v, st, a, cu = ref.inputs([1] * 5)
    x = [t[:, None] for t in (q, k, v)]
    out, ns = gdn.linear_decode.run(*x, None, a, None)
    ref.check(out[:, 0], ns, ref.reference(q, k, v, None, a, cu, SCALE), chunked=False)
    want = gdn.linear_decode.run(*x, st, a, SCALE)
    out = torch.empty_like(x[2])
    gdn.linear_decode.kernel(*x, st, a, SCALE, out, st)
    assert torch.equal(out, want[0]) and torch.equal(st, want[1])


def test_decode_forgets_at_minus_infinity():
    q, k, v, st, a, cu = ref.inputs([1] * 3)
    a[1] = -float("inf")
    out, ns = gdn.linear_decode.run(q[:, None], k[:, None], v[:, None], st, a, SCALE)
    ref.check(out[:, 0], ns, ref.reference(q, k, v, st, a, cu, SCALE), chunked=False)


@pytest.mark.parametrize("lens", [[1], [2], [63], [64], [65], [127, 1, 64], [0], [0, 5, 0, 130, 0], [200] * 3, [1] * 40,
                                  [512], [513], [700, 3], [1100], [1, 2000, 0, 33]])
@pytest.mark.parametrize("per_token", [False, True])
def test_prefill_lengths(lens, per_token):
    x = ref.inputs(lens, seed=len(lens), per_token=per_token)
    out, ns = _run(x)
    ref.check(out, ns, ref.reference(*x, SCALE), chunked=True)


@pytest.mark.parametrize("H,HV", [(1, 1), (16, 32), (3, 9), (8, 8), (2, 12), (1, 70)])
def test_prefill_heads(H, HV):
    x = ref.inputs([70, 1, 129], H, HV, seed=HV)
    out, ns = _run(x, torch.int64)
    ref.check(out, ns, ref.reference(*x, SCALE), chunked=True)


def test_prefill_long_and_cut_with_state_in_place():
    """Several segments for some sequences, one for others; the state written over its input."""
    x = ref.inputs([2500, 10, 0, 1300, 64], seed=3)
    want = ref.reference(*x, SCALE)
    q, k, v, st, a, cu = x
    out, ns = _run(x)
    ref.check(out, ns, want, chunked=True)
    for _ in range(3):
        st2, o2 = st.clone(), torch.empty_like(out)
        gdn.linear_prefill.kernel(q, k, v, st2, a, _cu(cu), SCALE, o2, st2)
        assert torch.equal(o2, out) and torch.equal(st2, ns)


@pytest.mark.parametrize("where", ["none", "zero", "strong", "minus_inf"])
def test_prefill_decays(where):
    x = ref.inputs([300, 77], seed=5)
    a = x[4]
    if where == "none":
        a[:] = 0
    elif where == "zero":
        a[100:140] = 0
    elif where == "strong":
        a[:] = a * 60
    else:
        a[::7] = -float("inf")
        a[64] = -float("inf")
    out, ns = _run(x)
    ref.check(out, ns, ref.reference(*x, SCALE), chunked=True)


def test_prefill_without_state_and_zero_tokens():
    x = list(ref.inputs([90, 0], with_state=False))
    out, ns = _run(x)
    ref.check(out, ns, ref.reference(*x, SCALE), chunked=True)
    assert not ns[1].any()
    q, k, v, st, a, cu = ref.inputs([0, 0])
    out, ns = gdn.linear_prefill.run(q, k, v, st, a, _cu(cu), SCALE)
    assert out.shape[0] == 0 and torch.equal(ns, st)


@pytest.mark.parametrize("lens", [[5], [100, 64], [30, 1000]])
def test_prefill_rows_outside_every_sequence(lens):
    """They may hold anything: no sequence reads them, `run` gives zeros there and `kernel` leaves them."""
    x = list(ref.inputs(lens, lead=3, tail=70))
    q, k, v, st, a, cu = x
    want = ref.reference(*x, SCALE)
    for t in (q, k, v, a):
        t[:3] = float("nan")
        t[cu[-1]:] = float("inf")
    out, ns = _run(x)
    assert not out[:3].any() and not out[cu[-1]:].any()
    ref.check(out, ns, want, chunked=True)
    o2 = torch.full_like(out, 7.0)
    gdn.linear_prefill.kernel(q, k, v, st, a, _cu(cu), SCALE, o2, torch.empty_like(ns))
    assert (o2[:3] == 7).all() and (o2[cu[-1]:] == 7).all() and torch.equal(o2[3:cu[-1]], out[3:cu[-1]])


def test_prefill_neighbours_do_not_reach_a_sequence():
    """The last chunk of a sequence ends inside a tile that also holds its neighbour's tokens."""
    x = list(ref.inputs([70, 60, 100], seed=2))
    q, k, v, st, a, cu = x
    want = ref.reference(*x, SCALE)
    for t in (q, k, v):
        t[70:130] = float("nan")
    out, ns = _run(x)
    keep = [0, 2]
    rows = torch.cat([torch.arange(70), torch.arange(130, 230)]).cuda()
    ref.check(out[rows], ns[keep], [want[0][rows], want[1][keep], want[2][rows], want[3][keep]], chunked=True)


def test_prefill_then_decode_is_one_longer_prefill():
    x = ref.inputs([131], seed=9)
    q, k, v, st, a, cu = x
    o1, s1 = gdn.linear_prefill.run(q[:130], k[:130], v[:130], st, a[:130], _cu([0, 130]), SCALE)
    o2, s2 = gdn.linear_decode.run(q[130:, None], k[130:, None], v[130:, None], s1, a[130:], SCALE)
    ref.check(torch.cat([o1, o2[:, 0]]), s2, ref.reference(*x, SCALE), chunked=True)


def test_prefill_strided_inputs_and_other_stream():
    x = ref.inputs([150, 20], seed=4)
    q, k, v, st, a, cu = x
    want = _run(x)
    wide = torch.cat([q, k, v], 1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = gdn.linear_prefill.run(wide[:, :4], wide[:, 4:8], wide[:, 8:], st, a, _cu(cu), SCALE)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_captured_and_replayed():
    """One graph of a prompt and a token, replayed on new inputs, gives the eager results bit for bit."""
    x = ref.inputs([700, 40], seed=6)
    q, k, v, st, a, cu = x
    cu_t = _cu(cu)
    n = len(cu) - 1
    out, ns, o1 = torch.empty_like(v), torch.empty_like(st), torch.empty_like(v[:n, None])
    ws = torch.empty(gdn.linear_prefill.workspace_bytes(n, q.shape[0]), dtype=torch.uint8, device="cuda")

    def step():
        gdn.linear_prefill.kernel(q, k, v, st, a, cu_t, SCALE, out, ns, workspace=ws)
        gdn.linear_decode.kernel(q[:n, None], k[:n, None], v[:n, None], ns, a[:n], SCALE, o1, ns)

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    y = ref.inputs([700, 40], seed=7)
    for dst, src in zip((q, k, v, st, a), y):
        dst.copy_(src)
    step()
    want = [t.clone() for t in (out, ns, o1)]
    for t in (out, ns, o1):
        t.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, w) for p, w in zip((out, ns, o1), want))
    assert gdn.linear_prefill.read_status(ws) == 0


def test_two_runs_are_bit_identical():
    x = ref.inputs([1500, 300], seed=8)
    a, b = _run(x), _run(x)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_overlapping_cu_seqlens_stays_in_bounds():
    """cu_seqlens that is not non-decreasing: results are invalid, but nothing outside the tensors is written."""
    q, k, v, st, a, _ = ref.inputs([1200, 0, 0])
    guard = torch.full((1200 + 64, 8, 128), 3.0, dtype=torch.bfloat16, device="cuda")
    cu = torch.tensor([0, 1200, 100, 5000], dtype=torch.int64, device="cuda")
    ns = torch.full((3 + 1, 8, 128, 128), 3.0, device="cuda")
    gdn.linear_prefill.kernel(q, k, v, st, a, cu, SCALE, guard[:1200], ns[:3])
    torch.cuda.synchronize()
    assert (guard[1200:] == 3).all() and (ns[3] == 3).all()
    x = ref.inputs([65])
    ref.check(*_run(x), ref.reference(*x, SCALE), chunked=True)


def test_refusals():
    q, k, v, st, a, cu = ref.inputs([10])
    c = _cu(cu)
    P, Dc = gdn.linear_prefill, gdn.linear_decode
    with pytest.raises(ValueError, match="log_decay"):
        P.run(q, k, v, st, a[:9], c, SCALE)
    with pytest.raises(ValueError, match="state"):
        P.run(q, k, v, st[:, :4], a, c, SCALE)
    with pytest.raises(ValueError, match="multiple"):
        P.run(q, k, v[:, :6], None, a[:, :6], c, SCALE)
    with pytest.raises(ValueError, match="int32 or int64"):
        P.run(q, k, v, st, a, c.float(), SCALE)
    with pytest.raises(ValueError, match="workspace"):
        P.kernel(q, k, v, st, a, c, SCALE, torch.empty_like(v), torch.empty_like(st),
                 workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(ValueError, match="output"):
        P.kernel(q, k, v, st, a, c, SCALE, v.float(), torch.empty_like(st))
    with pytest.raises(ValueError, match="new_state"):
        Dc.kernel(q[:1, None], k[:1, None], v[:1, None], st, a[:1], SCALE, torch.empty_like(v[:1, None]), st[:, :4])
    with pytest.raises(ValueError, match="must be \\["):
        Dc.run(q, k, v, st, a, SCALE)
    assert _lib.load().gdn_version() >= 100


@pytest.mark.parametrize("lens", [[700] * 17, [1100] * 3, [64, 1500] * 4, [1] * 3000, [0] * 50 + [2100]])
def test_many_and_equal_segments(lens):
    """Batches whose segments all stay whole beside ones that are cut, and searches over many sequences."""
    x = ref.inputs(lens, 1, 2, seed=len(lens))
    out, ns = _run(x)
    ref.check(out, ns, ref.reference(*x, SCALE), chunked=True)


def test_one_graph_for_other_lengths():
    """cu_seqlens may change between replays: one long sequence, two, and a short one beside a long one."""
    x = ref.inputs([3000, 0], seed=11)
    q, k, v, st, a, cu = x
    c, out, ns = _cu(cu), torch.empty_like(v), torch.empty_like(st)
    ws = torch.empty(gdn.linear_prefill.workspace_bytes(2, 3000, q.shape[1], v.shape[1]), dtype=torch.uint8, device="cuda")
    call = lambda: gdn.linear_prefill.kernel(q, k, v, st, a, c, SCALE, out, ns, workspace=ws)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for ends in ([0, 1500, 3000], [0, 3000, 3000], [0, 100, 3000], [0, 500, 1000]):
        c.copy_(_cu(ends))
        graph.replay()
        want = ref.reference(q, k, v, st, a, ends, SCALE)
        ref.check(out[:ends[-1]], ns, [w[:ends[-1]] if i in (0, 2) else w for i, w in enumerate(want)], chunked=True)
        assert gdn.linear_prefill.read_status(ws) == 0


@pytest.mark.parametrize("lens", [[], [0], [0, 0, 0]])
def test_no_token_belongs_to_a_sequence(lens):
    q, k, v, st, a, cu = ref.inputs(lens, tail=9)
    junk = torch.full((1 << 16,), float("nan"), device="cuda")  # freed memory that is not zero
    del junk
    out, ns = _run((q, k, v, st, a, cu))
    assert out.shape == v.shape and not out.any()
    assert torch.equal(ns, st)


def test_a_long_padded_tail_is_zeroed():
    x = list(ref.inputs([100, 30], lead=5, tail=5000))
    want = ref.reference(*x, SCALE)
    out, ns = _run(x)
    assert not out[:5].any() and not out[x[5][-1]:].any()
    ref.check(out, ns, want, chunked=True)


@pytest.mark.parametrize("with_state", [False, True])
def test_partial_chunks_beside_rows_that_are_not_finite(with_state):
    """Every CTA begins with a chunk whose tile also holds a neighbour's tokens, all of them NaN or infinite."""
    lens = [1 + 7 * i % 63 for i in range(600)]
    x = list(ref.inputs(lens, 1, 1, seed=12, with_state=with_state, tail=64))
    q, k, v, st, a, cu = x
    want = ref.reference(*x, SCALE)
    foreign = torch.ones(q.shape[0], dtype=torch.bool)
    for n in range(0, len(lens), 2):
        foreign[cu[n]:cu[n + 1]] = False
    for t, junk in ((q, float("nan")), (k, float("inf")), (v, float("nan"))):
        t[foreign.cuda()] = junk
    v[cu[1]:cu[2]] = float("inf")
    keep = (~foreign).cuda()
    for _ in range(20):
        out, ns = _run(x)
        ref.check(out[keep], ns[::2], [want[0][keep], want[1][::2], want[2][keep], want[3][::2]], chunked=True)


@pytest.mark.parametrize("N,T", [(3, 1200), (40, 2000), (65536, 1 << 22)])
def test_sequences_that_overlap_too_much_are_reported(N, T):
    """Every other sequence holds all tokens; the last size has 2^31 chunks.  Nothing is computed, in bounds and at once."""
    q, k, v = (torch.zeros((T, 1, 128), dtype=torch.bfloat16, device="cuda") for _ in range(3))
    out = torch.full_like(v, 3.0)
    ns = torch.empty((N, 1, 128, 128), device="cuda")
    ns[-1] = 3.0
    cu = torch.arange(N + 1, device="cuda") % 2 * T
    ws = torch.empty(gdn.linear_prefill.workspace_bytes(N, T, 1, 1), dtype=torch.uint8, device="cuda")
    gdn.linear_prefill.kernel(q, k, v, None, torch.zeros(1, device="cuda"), cu, SCALE, out, ns, workspace=ws)
    assert gdn.linear_prefill.read_status(ws) == 5
    assert (out[::997] == 3).all() and (ns[-1] == 3).all()
    gdn.linear_prefill.kernel(q, k, v, None, torch.zeros(1, device="cuda"), cu[:2], SCALE, out, ns[:1], workspace=ws)
    assert gdn.linear_prefill.read_status(ws) == 0 and not out.any() and not ns[0].any()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("lens,tokens", [([64], [0, 63]), ([64], [40]), ([100, 30], [10, 99, 115]), ([2500, 3], [1, 1300, 2400]),
                                         ([200] * 3, [63, 64, 300, 463, 599])])
def test_v_that_is_not_finite_reaches_later_tokens_only(bad, lens, tokens):
    """Its V column of the head, from its token on; the tokens before it in the same chunk keep their values."""
    x = ref.inputs(lens, 2, 4, seed=13)
    v = x[2]
    want = ref.reference(*x, SCALE)
    for i, t in enumerate(tokens):
        v[t, i % 4, 37 * i % 128] = bad
        v[t, i % 4, 127 - i] = bad
    dirty = ref.reference(*x, SCALE)
    out, ns = _run(x)
    for got, bad_ref in ((out, dirty[0]), (ns, dirty[1])):
        hit = ~torch.isfinite(bad_ref)
        assert torch.equal(~torch.isfinite(got.double()), hit) and hit.any()
    fill = lambda got, ref_, hit: torch.where(hit, ref_.to(got.dtype), got)  # noqa: E731
    ref.check(fill(out, want[0], ~torch.isfinite(dirty[0])), fill(ns, want[1], ~torch.isfinite(dirty[1])), want, chunked=True)


@pytest.mark.parametrize("what", ["q", "k", "decay", "state"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_what_is_not_finite_stays_where_it_belongs(what, bad):
    """q in its token, k and the decay from their token on, a state in its sequence and V rows."""
    if what == "decay":
        bad = float("nan")  # log decays are at most 0
    lens = [130, 64, 300]
    x = ref.inputs(lens, 2, 4, seed=14)
    q, k, v, st, a, cu = x
    want = ref.reference(*x, SCALE)
    if what == "state":
        st[1, 2, 17, 3] = bad
    else:
        t = {"q": q, "k": k, "decay": a}[what]
        for i in (40, 150, 194 + 64, 194 + 299):
            t[(i, 1, 5) if what != "decay" else (i, 1)] = bad
    dirty = ref.reference(*x, SCALE)
    out, ns = _run(x)
    hit = [~torch.isfinite(dirty[0]), ~torch.isfinite(dirty[1])]
    assert torch.equal(~torch.isfinite(out), hit[0]) and torch.equal(~torch.isfinite(ns), hit[1]) and hit[0].any()
    ref.check(torch.where(hit[0], want[0].to(out.dtype), out), torch.where(hit[1], want[1].float(), ns), want, chunked=True)


@pytest.mark.parametrize("HV", [1, 8])
def test_the_state_keeps_24_bits_of_a_decayed_v(HV):
    """Keys of one 1 each: every column of the state holds one decayed v, and no sum hides what it lost.

    The exponents stay below 1, so each of their sums is off by 2^-25 at most: some 30 of them, over two chunks, move a
    result by 30 * 2^-25 * ln 2 = 6.2e-7; two exponentials of 2^-22 each and four fp32 roundings of 2^-24 add 7.2e-7.
    That is below 2^-19 = 1.9e-6.  Two bf16 parts of the decayed v would be off by up to 2^-17 = 7.6e-6.
    """
    g = torch.Generator().manual_seed(15)
    k = torch.eye(128)[torch.randperm(128, generator=g)][:, None].to(torch.bfloat16).cuda()
    v = torch.randn((128, HV, 128), generator=g).to(torch.bfloat16).cuda()
    a = (-0.005 * torch.rand((128, HV), generator=g)).cuda()
    want = ref.reference(k, k, v, None, a, [0, 128], SCALE)
    _, ns = _run((k, k, v, None, a, [0, 128]))
    assert ((ns.double() - want[1]).abs() <= 2.0 ** -19 * want[1].abs()).all()
