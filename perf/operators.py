"""Cases of the linear-attention and 8-bit-cache operators: inputs, one pass, its work and its exact value.

Four operators, two families of token mixers:

* ``linear_prefill`` / ``linear_decode``: linear attention with a decay for each head over the k-last fp32 state
  [*, HV, V, K]: S' = e^a S + v k^T, o = scale S' q, for packed prompts and for single tokens;
* ``cache_append`` / ``cache_attend``: a paged key/value cache of 8-bit codes with one scale for each page and head,
  filled from bf16 rows and read by the attention of the last Q tokens of every sequence.

With ``own`` false, ``run`` computes them from elementary torch operations in fp32; with ``own`` true it calls ``gdn``.
"""
import math
import os
import sys

import torch

own = False

D = 128
_gdn = None


def _lib():
    global _gdn
    if _gdn is None:
        p = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gated-delta-network_b200")
        if p not in sys.path:
            sys.path.insert(0, p)
        import gdn

        _gdn = gdn
    return _gdn


# ---- cases ----------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one sequence generating a token: launch latency
        dict(name="linear_decode_b1", op="linear_decode", B=1, H=4, HV=8, per_token=False),
        # the benchmark's decode batch, gated per token
        dict(name="linear_decode_b64", op="linear_decode", B=64, H=4, HV=8, per_token=True),
        # a full serving batch of a 16 / 32-head layer
        dict(name="linear_decode_b250_h32", op="linear_decode", B=250, H=16, HV=32, per_token=True),
        # a short question: one sequence of a few tokens
        dict(name="linear_prefill_1x100", op="linear_prefill", N=1, lo=100, hi=100, H=4, HV=8, per_token=True),
        # one long prompt, the benchmark's 8192 tokens
        dict(name="linear_prefill_1x8192", op="linear_prefill", N=1, lo=8192, hi=8192, H=4, HV=8, per_token=False),
        # a ragged batch of prompts
        dict(name="linear_prefill_16_ragged", op="linear_prefill", N=16, lo=6, hi=8192, H=4, HV=8, per_token=True),
        # the benchmark's packed batch: many equal prompts, throughput
        dict(name="linear_prefill_64x4096", op="linear_prefill", N=64, lo=4096, hi=4096, H=4, HV=8, per_token=False),
        # one sequence, one token, a short history: launch latency
        dict(name="cache_attend_b1_1000", op="cache_attend", B=1, Q=1, Hq=32, Hkv=8, P=16, code="e4m3", lo=1000, hi=1000),
        # a serving batch at an ordinary length
        dict(name="cache_attend_b64_4096", op="cache_attend", B=64, Q=1, Hq=32, Hkv=8, P=64, code="e4m3", lo=4096,
             hi=4096),
        # a ragged batch up to long documents, four tokens verified at once
        dict(name="cache_attend_ragged_q4", op="cache_attend", B=24, Q=4, Hq=16, Hkv=2, P=32, code="int8", lo=1,
             hi=60000),
        # the new token of every sequence of a serving batch
        dict(name="cache_append_decode_b200", op="cache_append", B=200, Hkv=8, P=16, code="e4m3", lo=1, hi=1, past=1000),
        # the prompts of a ragged batch, some of them behind an earlier turn
        dict(name="cache_append_prompts", op="cache_append", B=12, Hkv=8, P=64, code="int8", lo=10, hi=8192, past=500),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear_decode", "linear_prefill", "cache_attend", "cache_append"])
    if op == "linear_decode":
        H, HV = rng.choice([(4, 8), (16, 32), (8, 8), (2, 12)])
        return dict(op=op, B=_log(rng, 1, 8000 // HV), H=H, HV=HV, per_token=rng.random() < 0.5)
    if op == "linear_prefill":
        H, HV = rng.choice([(4, 8), (16, 32), (8, 8), (3, 9)])
        N = _log(rng, 1, 64)
        hi = _log(rng, 1, min(8192, 2000000 // (N * HV)))
        lo = _log(rng, 1, hi)
        return dict(op=op, N=N, lo=lo, hi=hi, H=H, HV=HV, per_token=rng.random() < 0.5)
    code, P = rng.choice(["e4m3", "int8"]), rng.choice([16, 32, 64])
    if op == "cache_attend":
        Hq, Hkv = rng.choice([(32, 8), (16, 2), (8, 8), (12, 1)])
        B = _log(rng, 1, 128)
        hi = _log(rng, 10, min(60000, 2000000 // (B * Hkv)))
        lo = _log(rng, 1, hi)
        return dict(op=op, B=B, Q=rng.choice([1, 1, 2, 3, 5, 8]), Hq=Hq, Hkv=Hkv, P=P, code=code, lo=lo, hi=hi)
    B = _log(rng, 1, 256)
    hi = _log(rng, 1, min(8192, 16000 // B))
    return dict(op=op, B=B, Hkv=rng.choice([1, 2, 8]), P=P, code=code, lo=_log(rng, 1, hi), hi=hi,
                past=_log(rng, 1, 2000))


def _lens(n, lo, hi):
    """n lengths from lo to hi, evenly spread over their logarithm and out of order."""
    if n == 1:
        return [hi]
    step = next(s for s in (7, 5, 3, 1) if math.gcd(s, n) == 1)
    return [int(round(math.exp(math.log(lo) + (math.log(hi) - math.log(lo)) * ((i * step) % n) / (n - 1))))
            for i in range(n)]


def _work_lens(case):
    if case["op"] == "linear_prefill":
        return _lens(case["N"], case["lo"], case["hi"])
    return _lens(case["B"], case["lo"], case["hi"])


def work(case):
    op = case["op"]
    if op in ("linear_decode", "linear_prefill"):
        H, HV = case["H"], case["HV"]
        n = case["B"] if op == "linear_decode" else case["N"]
        T = n if op == "linear_decode" else sum(_work_lens(case))
        rows = T * (2 * H + 2 * HV) * D * 2 + (T if case["per_token"] else 1) * HV * 4
        return {"bytes": rows + 2 * n * HV * D * D * 4, "flops": 4 * T * HV * D * D}
    lens = _work_lens(case)
    if op == "cache_attend":
        B, Q, Hq, Hkv, P = (case[k] for k in ("B", "Q", "Hq", "Hkv", "P"))
        pages = sum((n + P - 1) // P for n in lens)
        return {"bytes": sum(lens) * Hkv * 2 * D + pages * (Hkv * 8 + 4) + 2 * B * Q * Hq * D * 2 + 4 * B,
                "flops": 4 * sum(lens) * Q * Hq * D}
    T = sum(lens)
    return {"bytes": T * case["Hkv"] * 2 * D * 3, "flops": 4 * T * case["Hkv"] * D}


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _rows(gen, *shape, unit=False):
    x = torch.randn(shape, generator=gen, device="cuda")
    if unit:
        x = x / x.square().sum(-1, keepdim=True).sqrt()
    return x.to(torch.bfloat16)


def _decay(gen, HV, tokens, per_token):
    """Log decays: a geometric range of horizons over the heads, gated per token where asked."""
    slope = -torch.exp2(-3.0 - 6.0 * torch.arange(HV, device="cuda") / HV)
    if not per_token:
        return slope
    return slope * (0.2 + 2.0 * torch.rand((*tokens, HV), generator=gen, device="cuda"))


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    op = case["op"]
    s = {"op": op}
    if op == "linear_decode":
        B, H, HV = case["B"], case["H"], case["HV"]
        s.update(q=_rows(gen, B, 1, H, D, unit=True), k=_rows(gen, B, 1, H, D, unit=True), v=_rows(gen, B, 1, HV, D),
                 state=torch.randn((B, HV, D, D), generator=gen, device="cuda") * 0.1,
                 decay=_decay(gen, HV, (B, 1), case["per_token"]), scale=D ** -0.5)
        return s
    lens = _work_lens(case)
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    T = cu[-1]
    if op == "linear_prefill":
        N, H, HV = case["N"], case["H"], case["HV"]
        s.update(q=_rows(gen, T, H, D, unit=True), k=_rows(gen, T, H, D, unit=True), v=_rows(gen, T, HV, D),
                 state=torch.randn((N, HV, D, D), generator=gen, device="cuda") * 0.1,
                 decay=_decay(gen, HV, (T,), case["per_token"]), scale=D ** -0.5, lens=lens,
                 cu=torch.tensor(cu, dtype=torch.int32, device="cuda"))
        return s
    B, Hkv, P = case["B"], case["Hkv"], case["P"]
    new = lens if op == "cache_append" else [0] * B
    past = [case["past"] + 37 * i % 97 for i in range(B)] if op == "cache_append" else lens
    total = [a + b for a, b in zip(past, new)]
    need = [(n + P - 1) // P for n in total]
    pages = sum(need)
    # every sequence's pages in an order of their own, as a server's free list hands them out
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    at = torch.arange(max(need), device="cuda")[None, :]
    first = torch.tensor([sum(need[:i]) for i in range(B)], device="cuda")[:, None]
    count = torch.tensor(need, device="cuda")[:, None]
    table = torch.where(at < count, order[(first + at).clamp(max=pages - 1)], torch.zeros_like(order[:1]))
    for name in ("k", "v"):
        x = torch.empty((pages, Hkv, P, D), dtype=torch.int8 if case["code"] == "int8" else torch.float8_e4m3fn,
                        device="cuda")
        for i in range(0, pages, 4096):  # a few pages at a time: the fp32 values of a whole cache are large
            r = torch.randn((min(4096, pages - i), Hkv, P, D), generator=gen, device="cuda")
            x[i:i + 4096] = ((r * 36.0).round().clamp(-127, 127) if case["code"] == "int8" else (r * 100.0).clamp(-448, 448)).to(x.dtype)
        s[name + "_cache"] = x
        unit = 1 / 36.0 if case["code"] == "int8" else 1 / 100.0
        s[name + "_scale"] = unit * (0.8 + 0.4 * torch.rand((pages, Hkv), generator=gen, device="cuda"))
    s.update(table=table.contiguous(), seq_lens=torch.tensor(total, dtype=torch.int32, device="cuda"), P=P)
    if op == "cache_attend":
        s.update(q=_rows(gen, B, case["Q"], case["Hq"], D), scale=D ** -0.5)
    else:
        s.update(k=_rows(gen, T, Hkv, D), v=_rows(gen, T, Hkv, D), cu=torch.tensor(cu, dtype=torch.int32, device="cuda"),
                 seq=torch.repeat_interleave(torch.arange(B, device="cuda"), torch.tensor(lens, device="cuda")))
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    g, op = _lib(), s["op"]
    if op == "linear_decode":
        return g.linear_decode.run(s["q"], s["k"], s["v"], s["state"], s["decay"], s["scale"])
    if op == "linear_prefill":
        return g.linear_prefill.run(s["q"], s["k"], s["v"], s["state"], s["decay"], s["cu"], s["scale"])
    if op == "cache_attend":
        return g.cache_attend.run(s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["table"],
                                  s["seq_lens"], s["scale"])
    g.cache_append.kernel(s["k"], s["v"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["table"],
                          s["seq_lens"], s["cu"])
    return s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]


def _run_plain(s):
    return {"linear_decode": _plain_decode, "linear_prefill": _plain_prefill, "cache_attend": _plain_attend,
            "cache_append": _plain_append}[s["op"]](s)


def _plain_decode(s):
    q, k, v = (s[n].float()[:, 0] for n in "qkv")
    group = v.shape[1] // q.shape[1]
    q, k = q.repeat_interleave(group, 1), k.repeat_interleave(group, 1)
    g = s["decay"].exp().reshape(-1, v.shape[1], 1, 1)
    state = s["state"] * g + v[..., :, None] * k[..., None, :]
    out = (state * q[..., None, :]).sum(-1) * s["scale"]
    return out[:, None].to(torch.bfloat16), state


def _plain_prefill(s, C=128):
    q, k, v, cu = s["q"], s["k"], s["v"], s["cu"].long()
    T, HV = v.shape[:2]
    N, group = cu.numel() - 1, HV // q.shape[1]
    n = (max(s["lens"]) + C - 1) // C
    # sequences padded to n chunks of C tokens; a padded token has k = v = 0 and no decay
    at = torch.arange(n * C, device=q.device)
    index = cu[:-1, None] + at
    inside = index < cu[1:, None]
    index = index.clamp(max=T - 1)

    def rows(x, times=1):
        x = x[index].float() * inside[..., None, None]
        return x.reshape(N, n, C, x.shape[2], D).permute(0, 1, 3, 2, 4).repeat_interleave(times, 2)

    qp, kp, vp = rows(q, group), rows(k, group), rows(v)
    a = s["decay"].double().expand(T, HV)[index] * inside[..., None]
    G = a.reshape(N, n, C, HV).permute(0, 1, 3, 2).cumsum(-1)  # [N, n, HV, C], 64 bits: long sums
    later = torch.ones((C, C), dtype=torch.bool, device=q.device).triu(1)
    decay = (G[..., :, None] - G[..., None, :]).masked_fill(later, -math.inf).exp().float()
    out = (qp @ kp.transpose(-1, -2) * decay) @ vp
    last = G[..., -1:]
    update = (vp * (last - G).exp().float()[..., None]).transpose(-1, -2) @ kp  # [N, n, HV, V, K]
    through = last.exp().float()[..., None]
    state = s["state"]
    starts = []
    for c in range(n):
        starts.append(state)
        state = state * through[:, c] + update[:, c]
    starts = torch.stack(starts, 1)
    out = s["scale"] * (out + (qp * G.exp().float()[..., None]) @ starts.transpose(-1, -2))
    out = out.permute(0, 1, 3, 2, 4).reshape(N, n * C, HV, D)
    return out[inside].to(torch.bfloat16), state


def _pages(cache, scale, table):
    """Pages of a table as fp32 values [B, Hkv, tokens, D]."""
    codes = cache.view(torch.uint8)[table].view(cache.dtype).float()
    x = codes * scale[table][..., None, None]
    B, n, Hkv, P, _ = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(B, Hkv, n * P, D)


def _plain_attend(s):
    table = s["table"].long()
    k, v = (_pages(s[n + "_cache"], s[n + "_scale"], table) for n in "kv")
    B, Q, Hq, _ = s["q"].shape
    Hkv, L = k.shape[1], k.shape[2]
    q = s["q"].float().reshape(B, Q, Hkv, Hq // Hkv, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, -1, D)
    w = (q @ k.transpose(-1, -2)) * s["scale"]
    seen = s["seq_lens"].long()[:, None] - Q + 1 + torch.arange(Q, device=w.device)  # tokens that row i sees
    hidden = torch.arange(L, device=w.device) >= seen[..., None]
    w = w.reshape(B, Hkv, Q, -1, L).masked_fill(hidden[:, None, :, None], -math.inf)
    w = (w - w.amax(-1, keepdim=True).clamp(min=-3e38)).exp()
    total = w.sum(-1, keepdim=True)
    w = (w / total.masked_fill(total == 0, 1)).reshape(B, Hkv, -1, L)
    out = (w @ v).reshape(B, Hkv, Q, -1, D).permute(0, 2, 1, 3, 4).reshape(B, Q, Hq, D)
    return out.to(torch.bfloat16)


def _encode(x, scale, dtype):
    """fp32 values to codes: x / scale, to the nearest (ties to even); a scale of zero gives zero."""
    y = torch.where(scale > 0, x / scale, torch.zeros_like(x))
    if dtype == torch.int8:
        return y.round().clamp(-127, 127).to(torch.int8)
    return y.clamp(-448, 448).to(dtype)


def _plain_append(s):
    table, cu, seq, P = s["table"].long(), s["cu"].long(), s["seq"], s["P"]
    T = s["k"].shape[0]
    start = s["seq_lens"].long() - (cu[1:] - cu[:-1])
    at = start[seq] + torch.arange(T, device=cu.device) - cu[:-1][seq]
    page, slot = table[seq, at // P], at % P
    # the first page that a sequence writes may hold older tokens; the others are begun by this call
    head, held = table.gather(1, (start // P)[:, None])[:, 0], start % P
    out = []
    for name in "kv":
        x, cache, scale = s[name].float(), s[name + "_cache"], s[name + "_scale"]
        limit = torch.full((), 127.0 if cache.dtype == torch.int8 else 448.0, device=x.device)
        top = x.abs().amax(-1) / limit  # [T, Hkv]
        old = scale[head]
        begun = torch.where((held == 0)[:, None], torch.zeros_like(old), old)
        scale[page] = 0
        scale[head] = begun
        scale.index_reduce_(0, page, top, "amax")
        new = scale[head]
        raw = cache.view(torch.uint8)
        codes = raw[head].view(cache.dtype)
        again = _encode(codes.float() * old[..., None, None], new[..., None, None], cache.dtype)
        kept = (torch.arange(P, device=x.device) < held[:, None])[:, None, :, None] & (new > old)[..., None, None]
        raw[head] = torch.where(kept, again.view(torch.uint8), codes.view(torch.uint8))
        raw[page, :, slot] = _encode(x, scale[page][..., None], cache.dtype).view(torch.uint8)
        out.append(cache)
    return out[0], out[1], s["k_scale"], s["v_scale"]


# ---- 64 bits --------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"linear_decode": _exact_linear, "linear_prefill": _exact_linear, "cache_attend": _exact_attend,
            "cache_append": _exact_append}[s["op"]](s)


def _exact_linear(s):
    """Token by token, all sequences abreast."""
    one = s["op"] == "linear_decode"
    lens = [1] * s["q"].shape[0] if one else s["lens"]
    q, k, v = (s[n].reshape(-1, *s[n].shape[-2:]) for n in "qkv")
    HV = v.shape[1]
    group = HV // q.shape[1]
    a = s["decay"].reshape(-1, HV).expand(v.shape[0], HV)
    state = s["state"].double()
    out = torch.zeros(v.shape, dtype=torch.float64, device=v.device)
    # sequences from the longest down, so that the running ones come first
    order = sorted(range(len(lens)), key=lambda i: -lens[i])
    base = [sum(lens[:i]) for i in range(len(lens))]
    first = torch.tensor([base[i] for i in order], device=v.device)
    state = state[torch.tensor(order, device=v.device)].clone()
    running = len(order)
    for t in range(max(lens)):
        while lens[order[running - 1]] <= t:
            running -= 1
        at = first[:running] + t
        now = state[:running]
        now.mul_(a[at].double().exp()[..., None, None])
        kt = k[at].double().repeat_interleave(group, 1)
        qt = q[at].double().repeat_interleave(group, 1)
        now.add_(v[at].double()[..., :, None] * kt[..., None, :])
        out[at] = s["scale"] * torch.matmul(now, qt[..., None])[..., 0]
    final = torch.empty_like(state)
    final[torch.tensor(order, device=v.device)] = state
    return (out[:, None] if one else out), final


def _exact_attend(s):
    B, Q, Hq, _ = s["q"].shape
    P, Hkv = s["P"], s["k_cache"].shape[1]
    out = torch.zeros((B, Q, Hq, D), dtype=torch.float64, device=s["q"].device)
    for b, n in enumerate(s["seq_lens"].tolist()):
        pages = s["table"][b, : (n + P - 1) // P].long()
        for h in range(Hkv):
            kv = []
            for name in "kv":
                codes = s[name + "_cache"].view(torch.uint8)[pages, h].view(s[name + "_cache"].dtype).double()
                kv.append((codes * s[name + "_scale"][pages, h].double()[:, None, None]).reshape(-1, D)[:n])
            heads = slice(h * (Hq // Hkv), (h + 1) * (Hq // Hkv))
            for i in range(Q):
                m = n - Q + 1 + i
                if m > 0:
                    w = torch.softmax(s["scale"] * (s["q"][b, i, heads].double() @ kv[0][:m].T), -1)
                    out[b, i, heads] = w @ kv[1][:m]
    return out


def _exact_append(s):
    """Page by page; codes of whole numbers have no value between two of them, so they are left out."""
    P, res = s["P"], []
    cu, total, table = s["cu"].tolist(), s["seq_lens"].tolist(), s["table"].tolist()
    integer = s["k_cache"].dtype == torch.int8
    top = 127.0 if integer else 448.0
    scales = []
    for name in "kv":
        cache = None if integer else s[name + "_cache"].to(torch.float64)
        scale = s[name + "_scale"].double()
        for b in range(len(total)):
            x = s[name][cu[b]:cu[b + 1]].double()
            begin = total[b] - x.shape[0]
            p = begin // P
            while p * P < total[b]:
                lo, hi = max(begin, p * P), min(total[b], (p + 1) * P)
                part, id_ = x[lo - begin:hi - begin], table[b][p]
                was = scale[id_] if lo > p * P else torch.zeros_like(scale[id_])
                to = torch.maximum(was, part.abs().amax((0, 2)) / top)
                if not integer:
                    if lo > p * P:
                        held = cache[id_, :, : lo - p * P]
                        moved = (held * (was / to)[:, None, None]).float().to(torch.float8_e4m3fn).double()
                        cache[id_, :, : lo - p * P] = torch.where((to > was)[:, None, None], moved, held)
                    put = (part / to[:, None]).clamp(-448, 448).float().to(torch.float8_e4m3fn).double()
                    cache[id_, :, lo - p * P:hi - p * P] = put.transpose(0, 1)
                scale[id_] = to
                p += 1
        res.append(cache)
        scales.append(scale)
    return res[0], res[1], scales[0], scales[1]
