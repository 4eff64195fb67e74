"""Plain 64-bit restatement of the KV-cache operators (test infrastructure): the 8-bit block format, rotation and append, attention over a
slot's rows behind a shared prefix, and how far a 16-bit kernel may be from it."""
import math

import torch


def top(dtype):
    return 1.875 * 2.0 ** (15 if dtype == torch.float16 else 127)


def mx_encode(x, limit):
    """[..., D] 16-bit values -> (e4m3 bytes, scale bytes): block maximum, smallest power of two that brings it to 448, rounding to even."""
    fin = torch.isfinite(x)
    y = torch.where(fin, x.double(), torch.zeros((), dtype=torch.float64)).clamp(-limit, limit).unflatten(-1, (-1, 32))
    amax = y.abs().amax(-1, keepdim=True)
    e = torch.full_like(amax, -126.0)
    big = amax > 448.0 * 2.0 ** -126
    e[big] = torch.ceil(torch.log2(amax[big] / 448.0))
    e = torch.where(amax > 448.0 * torch.exp2(e), e + 1, e)                        # (log2 may round a power of two either way)
    e = torch.where((amax <= 448.0 * torch.exp2(e - 1)) & (e > -126), e - 1, e)
    y = (y / torch.exp2(e)).flatten(-2)
    mag = y.abs()
    step = torch.exp2(torch.floor(torch.log2(mag.clamp(min=2.0 ** -6))) - 3)
    k = torch.round(mag / step) * step                                             # on the e4m3 grid
    ex = torch.floor(torch.log2(k.clamp(min=2.0 ** -6)))
    sub = k < 2.0 ** -6
    code = torch.where(sub, k * 2.0 ** 9, (ex + 7) * 8 + (k / torch.exp2(ex) - 1) * 8).to(torch.int64)
    code = code + torch.where(torch.signbit(x.double()), 128, 0)
    code = torch.where(fin, code, torch.full_like(code, 127))
    return code.to(torch.uint8), (e.squeeze(-1) + 127).to(torch.uint8)


def mx_decode(code, scale):
    b = code.to(torch.int64)
    ex, man = (b >> 3) & 15, (b & 7).double()
    y = torch.where(ex == 0, man * 2.0 ** -9, (8 + man) * torch.exp2((ex - 10).double()))
    y = torch.where((b & 127) == 127, torch.full_like(y, float("nan")), y)
    return torch.where(b >= 128, -y, y) * torch.exp2(scale.double() - 127).repeat_interleave(32, -1)


def rope(x, cos, sin):
    """x [..., D] in the 16-bit type, every product and the sum rounded to it."""
    dt, D = x.dtype, x.shape[-1]
    x = x.double()
    rot = torch.cat((-x[..., D // 2:], x[..., :D // 2]), -1)
    r = lambda t: t.to(torch.float32).to(dt).double()  # noqa: E731 - (products of two 16-bit values are exact in 32 bits)
    return r(r(x * cos.double()) + r(rot * sin.double())).to(dt)


def attention(q, keys, values, scale, causal, tokens):
    """One (slot, head): q [T, D], keys / values [P + n, D] with the slot's own n rows last, ``keys`` a pair (prefix rows P, all rows).
    Returns (out, tol): the result in 64 bits, zeros where a query sees nothing, and the bound on a kernel's distance from it that counts
    its roundings: output and probabilities to 16 bits (u each), fp32 scores (D + 16 roundings of the sum of magnitudes), exponential and
    sums (2^-19 and 2 n 2^-24 relative)."""
    P, k = keys
    v = values
    T, n = q.shape[0], k.shape[0] - P
    u = torch.finfo(q.dtype).eps / 2
    q, k, v = q.double(), k.double(), v.double()
    seen = torch.ones(T, P + n, dtype=torch.bool, device=q.device)
    if causal:
        seen[:, P:] = torch.arange(n, device=q.device) <= (n - T + torch.arange(T, device=q.device)).unsqueeze(1)
    s = torch.where(seen, scale * (q @ k.T), torch.full((), -math.inf, dtype=torch.float64, device=q.device))
    if P + n == 0:
        z = torch.zeros_like(q)
        return z, z
    m = s.amax(-1, keepdim=True)
    p = torch.where(seen, torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m)), torch.zeros_like(s))
    total = p.sum(-1, keepdim=True)
    total = torch.where(total == 0, torch.ones_like(total), total)
    out = torch.zeros_like(q)
    mean = torch.zeros_like(q)
    for t in range(T):                                                             # a row that a query does not see has no part in it
        w = p[t][seen[t]] / total[t]
        out[t] = w @ v[seen[t]]
        mean[t] = w @ v[seen[t]].abs()
    mags = scale * (q.abs() @ k.abs().T)
    worst = torch.where(seen, mags, torch.zeros_like(mags)).amax(-1, keepdim=True)
    D = q.shape[1]
    rel = 1.02 * u + 2 * ((D + 16) * 2.0 ** -24 * worst + 2.0 ** -20) + 2 * (P + n) * 2.0 ** -24
    floor = 2.0 ** -25 if u == 2.0 ** -11 else 0.0                                  # half of fp16's smallest subnormal: outputs ...
    tol = 1.01 * u * out.abs() + rel * mean + floor
    if floor:                                                                      # ... and probabilities, an absolute step each
        big = torch.stack([v[seen[t]].abs().sum(0) if bool(seen[t].any()) else torch.zeros(D, dtype=torch.float64, device=v.device) for t in range(T)])
        tol = tol + floor * big / total
    return out, tol
