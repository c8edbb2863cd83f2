"""The 8-bit paged cache: appending as the definition says (numpy fp32, so codes compare bit for bit) and attention in 64 bits."""
from __future__ import annotations

import numpy as np
import torch

D = 128
DTYPES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def empty_cache(pages, Hkv, P, code, device="cuda", seed=0):
    """A cache whose unwritten slots hold rubbish: every code pattern (NaN among the e4m3 ones), NaN scales."""
    g = torch.Generator().manual_seed(seed)
    raw = [torch.randint(0, 256, (pages, Hkv, P, D), generator=g, dtype=torch.uint8) for _ in range(2)]
    kc, vc = (x.to(device).view(DTYPES[code]) for x in raw)
    ks, vs = (torch.full((pages, Hkv), float("nan"), device=device) for _ in range(2))
    return kc, vc, ks, vs


def tables(lens, P, max_pages=None, seed=0, device="cuda", spare=3):
    """(block table of pages in a random order, page count); unused entries point far outside the cache."""
    need = [(n + P - 1) // P for n in lens]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    width = max(max(need, default=0), 1) if max_pages is None else max_pages
    t = torch.full((len(lens), width), 1 << 30, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        t[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    return t.to(device), pages


def encode(x, s, code):
    with np.errstate(all="ignore"):
        y = (x / s).astype(np.float32) if s > 0 else np.zeros_like(x)
    if code == "int8":
        return np.clip(np.rint(np.nan_to_num(y, nan=0.0, posinf=1e9, neginf=-1e9)), -127, 127).astype(np.int8).view(np.uint8)
    y = torch.from_numpy(np.clip(y, -448, 448))
    return y.to(torch.float8_e4m3fn).view(torch.uint8).numpy()


def decode(raw, code):
    t = torch.from_numpy(np.ascontiguousarray(raw))
    return (t.view(torch.int8) if code == "int8" else t.view(torch.float8_e4m3fn)).float().numpy()


def append(x, cache, scale, table, seq_lens, cu, code):
    """Expected (codes uint8, scales) after appending rows x [T, Hkv, 128] (CPU float32) to a cache on the GPU or CPU."""
    raw, sc = cache.view(torch.uint8).cpu().numpy().copy(), scale.cpu().numpy().copy()
    pages, Hkv, P, _ = raw.shape
    table = table.cpu().numpy()
    x = x.float().cpu().numpy()
    m = np.float32(127 if code == "int8" else 448)
    for b, end in enumerate(seq_lens):
        n = cu[b + 1] - cu[b]
        start = end - n
        for i in range(max(start, 0) // P, min((end + P - 1) // P, table.shape[1])):
            lo, hi = max(start, 0, i * P), min(end, (i + 1) * P)
            page = table[b, i]
            if lo >= hi or not 0 <= page < pages:
                continue
            for h in range(Hkv):
                part = x[cu[b] + lo - start:cu[b] + hi - start, h]
                mag = np.where(np.isfinite(part), np.abs(part), 0)
                old = sc[page, h] if lo > i * P else np.float32(0)
                s = max(old, np.float32(mag.max()) / m)
                if lo > i * P and s > old:
                    held = decode(raw[page, h, : lo - i * P], code)
                    raw[page, h, : lo - i * P] = encode((held * old).astype(np.float32), s, code)
                raw[page, h, lo - i * P:hi - i * P] = encode(part, s, code)
                sc[page, h] = s
    return raw, sc


def attend(q, kc, vc, ks, vs, table, seq_lens, scale):
    """(out [B,Q,Hq,128] float64, bound on the error of every element).

    The bound adds up the roundings: the bf16 output, 2^-8 of it; the weights in fp16, 2^-11 of each (2^-10 with the
    quotient of the value scales), or 2^-25 of the largest value scale where a weight is below fp16's normal range;
    the scores: 128 fp32 sums (2^-17 of the terms' magnitudes), q in fp16 with a power of two (2^-24 of its largest
    element times sum |k|), and the exponential's argument (2^-22 of it).
    """
    B, Q, Hq, _ = q.shape
    pages, Hkv, P, _ = kc.shape
    G = Hq // Hkv
    out = torch.zeros((B, Q, Hq, D), dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    for b, n in enumerate(seq_lens):
        n = min(n, table.shape[1] * P)
        idx = table[b, : (n + P - 1) // P].long()
        for h in range(Hkv):
            if n == 0:
                continue
            k, v = ((c.view(torch.uint8)[idx, h].view(c.dtype).double() * s[idx, h].double()[:, None, None]).reshape(-1, D)[:n]
                    for c, s in ((kc, ks), (vc, vs)))
            for i in range(Q):
                m = n - Q + 1 + i
                if m <= 0:
                    continue
                qq = q[b, i, h * G:(h + 1) * G].double()
                s = scale * (qq @ k[:m].T)
                w = torch.softmax(s, -1)
                d = abs(scale) * (2.0 ** -17 * (qq.abs() @ k[:m].abs().T)
                                  + 2.0 ** -24 * qq.abs().amax(-1, keepdim=True) * k[:m].abs().sum(-1)) + 2.0 ** -21 * s.abs()
                o = w @ v[:m]
                out[b, i, h * G:(h + 1) * G] = o
                tol[b, i, h * G:(h + 1) * G] = (2.0 ** -8 * o.abs() + (2.0 ** -10 + 2 * d.amax(-1, keepdim=True)) * (w @ v[:m].abs())
                                                + m * 2.0 ** -25 * v[:m].abs().amax() + 1e-30)
    return out, tol
