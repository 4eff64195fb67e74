"""KV caches by handle on the GPU: rows written, read back and attended to, against the 64-bit restatement in tests/_kv_ref.py (bit for bit
where the format decides, within the bound that _kv_ref.attention derives where sums do)."""
import math

import pytest
import torch

from seed_amd import lib as L
from seed_amd.kv_cache import KVAttention, KVCache
from tests import _kv_ref as R

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _rand(shape, dtype, seed, gain=1.0):
    return (torch.randn(shape, generator=_gen(seed)) * gain).to(dtype)


def _tables(rows, dim, dtype):
    ang = torch.arange(rows).double().unsqueeze(1) / 10000.0 ** (torch.arange(0, dim, 2).double() / dim)
    return tuple(torch.cat((f, f), -1).to(dtype) for f in (ang.cos(), ang.sin()))


def _poisoned(slots, heads, rows, dim, fmt, dtype):
    """A cache whose every byte reads as NaN."""
    if fmt == "16":
        k, v = (torch.full((slots, heads, rows, dim), float("nan"), dtype=dtype).cuda() for _ in range(2))
        return KVCache.wrap(k, v)
    k, v = (torch.full((slots, heads, rows, dim), 0x7F, dtype=torch.uint8).cuda() for _ in range(2))
    ks, vs = (torch.full((slots, heads, rows, dim // 32), 200, dtype=torch.uint8).cuda() for _ in range(2))
    return KVCache.wrap(k, v, ks, vs, dtype=dtype)


def _fill(cache, s, n, seed, gain=1.0, first=0):
    """Random rows first .. first + n - 1 of slot s; returns their values in 64 bits, [heads, n, dim] each."""
    shape = (cache.kv_heads, n, cache.head_dim)
    out = []
    for i, (rows, sc) in enumerate(((cache.k, cache.k_scale), (cache.v, cache.v_scale))):
        x = _rand(shape, cache.dtype, seed + i, gain)
        if cache.format == "16":
            rows[s, :, first:first + n] = x.cuda()
            out.append(x.double())
        else:
            code, byte = R.mx_encode(x, R.top(cache.dtype))
            rows[s, :, first:first + n] = code.cuda()
            sc[s, :, first:first + n] = byte.cuda()
            out.append(R.mx_decode(code, byte))
    return out


def _check(got, q, per_slot, prefix, heads, kv_heads, tokens, scale, causal, tag=""):
    """got [B*T, H*D] against the reference, slot by slot and head by head."""
    B = len(per_slot)
    D = q.shape[1] // heads
    got = got.cpu().double().view(B, tokens, heads, D)
    q = q.cpu().view(B, tokens, heads, D)
    for b, (k, v) in enumerate(per_slot):
        for h in range(heads):
            g = h // (heads // kv_heads)
            kk, vv = k[g], v[g]
            if prefix is not None:
                kk, vv = torch.cat((prefix[0][g], kk)), torch.cat((prefix[1][g], vv))
            P = 0 if prefix is None else prefix[0].shape[1]
            want, tol = R.attention(q[b, :, h], (P, kk), vv, scale, causal, tokens)
            off = (got[b, :, h] - want).abs()
            assert torch.isfinite(got[b, :, h]).all(), (tag, b, h)
            assert (off <= tol).all(), (tag, b, h, (off - tol).max().item(), off.max().item())


# ------------------------------------------------------------------------------------------------ append and read
@pytest.mark.parametrize("fmt", ["mx8", "16"])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("H,G,D,T,past", [(2, 2, 128, 1, [0, 5, 30]), (8, 2, 64, 7, [0, 3, 25]), (5, 1, 128, 33, [0, 1, 0]), (3, 3, 64, 1, [31, 30, -1]),
                                          (40, 40, 128, 2, [29, 31, 30])])
def test_append_is_the_formula_bit_for_bit(fmt, dtype, H, G, D, T, past):
    rows, B = 33, len(past)
    cache = _poisoned(B, G, rows, D, fmt, dtype)
    before = [t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale) if t is not None]
    cols = (H + 2 * G) * D
    wide = _rand((B * T, cols + 64), dtype, 7, 3.0).cuda()
    qkv = wide[:, 8:8 + cols]                                                      # a row stride of its own
    cos, sin = _tables(64, D, dtype)
    q_wide = torch.full((B * T, H * D + 8), 5.0, dtype=dtype).cuda()
    q = cache.append(qkv, cos.cuda(), sin.cuda(), torch.tensor(past, dtype=torch.int32).cuda(), heads=H, pos_base=9, q_out=q_wide[:, :H * D])
    torch.cuda.synchronize()
    assert (q_wide[:, H * D:] == 5.0).all()
    x = qkv.cpu().view(B, T, H + 2 * G, D)
    at = (torch.tensor(past).unsqueeze(1) + torch.arange(T) + 9).clamp(0, 63)
    rot = R.rope(x[:, :, :H + G], cos[at].unsqueeze(2), sin[at].unsqueeze(2))
    assert torch.equal(q.cpu().view(B, T, H, D), rot[:, :, :H])
    want = [t.cpu().clone() for t in before]
    for b in range(B):
        for t in range(T):
            r = past[b] + t
            if past[b] < 0 or r >= rows:
                continue
            k, v = rot[b, t, H:], x[b, t, H + G:]
            if fmt == "16":
                want[0][b, :, r], want[1][b, :, r] = k, v
            else:
                (want[0][b, :, r], want[2][b, :, r]), (want[1][b, :, r], want[3][b, :, r]) = R.mx_encode(k, R.top(dtype)), R.mx_encode(v, R.top(dtype))
    for w, got in zip(want, [t for t in (cache.k, cache.v, cache.k_scale, cache.v_scale) if t is not None]):
        assert torch.equal(w.view(torch.uint8), got.cpu().view(torch.uint8))      # rows that were not written keep their bytes


@pytest.mark.parametrize("dtype", [BF, HF])
def test_append_agrees_with_the_static_cache_kernel(dtype):
    """One layout, one length for all slots: the 16-bit handle writes what seedmi_rope_kv_append writes."""
    B, T, H, D, rows, past = 3, 4, 2, 128, 16, 5
    lib = L.load(dtype)
    qkv = _rand((B * T, 3 * H * D), dtype, 3).cuda()
    cos, sin = (t.cuda() for t in _tables(32, D, dtype))
    pos = torch.randint(0, 32, (B * T,), generator=_gen(4)).cuda()
    kc, vc = (torch.zeros(B, H, rows, D, dtype=dtype).cuda() for _ in range(2))
    q0 = torch.empty(B * T, H * D, dtype=dtype).cuda()
    L.check(lib.seedmi_rope_kv_append(L.ptr(qkv), 3 * H * D, L.ptr(pos), L.ptr(cos), L.ptr(sin), L.ptr(q0), H * D, L.ptr(kc), L.ptr(vc), B, T, H, D,
                                      rows, past, None, 32, L.stream_ptr()), "append", lib)
    cache = KVCache.new(B, H, rows, D, "16", dtype)
    q1 = cache.append(qkv, cos, sin, past, heads=H, pos_ids=pos)
    assert torch.equal(vc, cache.v)
    for a, b in ((q0, q1), (kc, cache.k)):
        if dtype == BF:
            assert torch.equal(a, b)
        else:
            # the fp16 build of seedmi_rope_kv_append adds one product unrounded (v_fma_f16): the sums differ by that product's rounding,
            # at most u |x| (|cos|, |sin| <= 1), and each is then rounded, at most u |sum| <= u sqrt(2) max|x| each
            u, big = 2.0 ** -11, qkv.abs().max().item()
            assert (a.double() - b.double()).abs().max().item() <= u * big * (1 + 2 * math.sqrt(2) * (1 + u))


@pytest.mark.parametrize("dtype", [BF, HF])
def test_special_values_of_the_8_bit_rows(dtype):
    """Blocks of zeros, of the type's largest and smallest values, with infinities and NaN: codes and scale bytes by the formula, finite
    values finite when read back."""
    D, fi = 128, torch.finfo(dtype)
    v = _rand((7, D), dtype, 1)
    v[0] = 0.0
    v[1] = fi.max
    v[1, ::3] = -fi.max
    v[2] = fi.tiny
    v[2, 5] = fi.smallest_normal * 3
    v[3, 7], v[3, 40], v[3, 41], v[3, 90] = float("inf"), float("-inf"), float("nan"), float("inf")
    v[4, 32:64] = float("nan")
    v[5] = torch.tensor([448.0, 449.0, -450.0, 1.75, 0.5, 2.0 ** -10, 2.0 ** -9, -0.0]).to(dtype).repeat(16)
    v[6, :32] = torch.tensor([1.75]).to(dtype) * 2.0
    cache = KVCache.new(1, 1, 8, D, "mx8", dtype)
    qkv = torch.cat((torch.zeros(7, 2 * D, dtype=dtype), v), 1).cuda()
    cos, sin = (t.cuda() for t in _tables(8, D, dtype))
    cache.append(qkv, cos, sin, 0, heads=1)
    code, byte = R.mx_encode(v, R.top(dtype))
    assert torch.equal(cache.v_scale[0, 0, :7].cpu(), byte)
    nan = (code & 127) == 127
    got = cache.v[0, 0, :7].cpu()
    assert torch.equal(got[~nan], code[~nan]) and ((got[nan] & 127) == 127).all()
    assert ((cache.k[0, 0] & 127) == 0).all() and (cache.k_scale[0, 0] == 1).all()  # (0 times a negative cosine is -0, as is -0 + -0)
    _, back = cache.read(0, 7)
    want = R.mx_decode(code, byte)
    assert torch.equal(torch.nan_to_num(back[0, 0].cpu().double(), nan=77.0), torch.nan_to_num(want.to(dtype).double(), nan=77.0))
    assert torch.isfinite(back[0, 0].cpu()[torch.isfinite(v)]).all()


@pytest.mark.parametrize("dtype,D,G,n", [(BF, 128, 3, 9), (HF, 64, 2, 1), (HF, 128, 1, 17), (BF, 64, 5, 4)])
def test_read_rows_of_every_slot(dtype, D, G, n):
    B, rows = 4, 20
    cache = _poisoned(B, G, rows, D, "mx8", dtype)
    vals = [_fill(cache, b, rows, 10 * b) for b in range(B)]
    starts = [0, 3, 14, -2]
    k, v = cache.read(torch.tensor(starts, dtype=torch.int32).cuda(), n)
    for got, i in ((k, 0), (v, 1)):
        want = torch.zeros(B, G, n, D, dtype=torch.float64)
        for b, s in enumerate(starts):
            for t in range(n):
                if 0 <= s + t < rows:
                    want[b, :, t] = vals[b][i][:, s + t]
        assert torch.equal(got.cpu().double(), want)
    k1, v1 = cache.read(2, n, slots=2)
    assert torch.equal(k1.cpu().double(), torch.stack([vals[b][0][:, 2:2 + n] for b in range(2)]))
    assert torch.equal(v1.cpu().double(), torch.stack([vals[b][1][:, 2:2 + n] for b in range(2)]))


def test_every_code_reads_back():
    """All 256 codes under scale bytes from the smallest to the largest that the formats produce."""
    for dtype, bytes_ in ((BF, [1, 100, 127, 200, 247]), (HF, [119, 120, 127, 134])):
        cache = KVCache.new(1, 1, 2 * len(bytes_), 128, "mx8", dtype)
        code = torch.arange(256, dtype=torch.uint8).view(2, 128).repeat(len(bytes_), 1)
        byte = torch.tensor(bytes_, dtype=torch.uint8).repeat_interleave(2).view(-1, 1).repeat(1, 4)
        cache.k[0, 0], cache.k_scale[0, 0] = code.cuda(), byte.cuda()
        k, _ = cache.read(0, 2 * len(bytes_))
        want = R.mx_decode(code, byte).to(torch.float32)
        want = want.to(dtype).double()
        got = k[0, 0].cpu().double()
        keep = torch.isfinite(want)
        if dtype == BF:                                                            # 2^-126 * 2^-9 lies below bf16's normal range
            keep &= (want.abs() >= 2.0 ** -126) | (want == 0)
        assert torch.equal(got[keep], want[keep])
        assert torch.isnan(got[torch.isnan(want)]).all()


# ------------------------------------------------------------------------------------------------ attention
CASES = [  # H, G, D, T, lengths, prefix, causal
    (2, 2, 128, 1, [1, 2, 31, 32, 33, 64, 65, 127, 128, 129, 0, 200], 0, True),
    (2, 2, 64, 1, [1, 63, 64, 130, 0], 0, True),
    (8, 2, 128, 1, [5, 190, 64], 0, True),
    (40, 40, 128, 1, [77, 1], 0, True),
    (12, 1, 64, 3, [3, 50, 2, 0, 129], 0, True),                                   # fewer rows than query tokens: the first see nothing
    (4, 4, 128, 5, [5, 37, 200], 0, True),
    (10, 2, 128, 17, [17, 18, 100, 9], 0, True),
    (3, 3, 128, 33, [33, 150, 1], 0, True),
    (4, 2, 64, 70, [70, 71, 199, 64], 0, True),
    (4, 4, 128, 130, [130, 200], 0, True),
    (6, 2, 128, 150, [150, 160, 40], 0, True),
    (2, 1, 128, 9, [40, 1, 0], 0, False),
    (2, 2, 64, 140, [33, 200, 0], 0, False),
    (2, 2, 128, 1, [1, 0, 40], 1, True),
    (4, 4, 128, 1, [3, 20, 0, 65], 100, True),
    (8, 2, 64, 1, [3, 20, 0, 65, 12, 1, 1], 65, True),
    (6, 2, 128, 4, [4, 30, 2, 65], 33, True),
    (5, 1, 128, 20, [20, 64], 64, True),
    (2, 2, 128, 140, [140, 150], 77, True),
    (4, 2, 64, 131, [131, 20], 129, True),
    (4, 4, 128, 64, [64, 200, 30], 0, True),
    (12, 4, 64, 27, [27, 64, 3], 65, True),
    (8, 2, 128, 100, [100, 164, 64], 0, True),
    (3, 1, 128, 171, [171, 172], 0, True),
]


@pytest.mark.parametrize("fmt,dtype", [("mx8", BF), ("mx8", HF), ("16", BF), ("16", HF)])
@pytest.mark.parametrize("H,G,D,T,lens,P,causal", CASES)
def test_attention_against_the_formula(fmt, dtype, H, G, D, T, lens, P, causal):
    B, rows = len(lens), 200
    cache = _poisoned(B, G, rows, D, fmt, dtype)
    per_slot = [[x[:, :n] for x in _fill(cache, b, max(n, 1), 100 * b + 1, 2.0)] for b, n in enumerate(lens)]
    for b, n in enumerate(lens):
        if n == 0:                                                                 # an idle slot's row is poison too
            cache.k[b].view(torch.uint8).fill_(0x7F)
            cache.v[b].view(torch.uint8).fill_(0xFF)
    prefix, vals = None, None
    if P:
        prefix = _poisoned(1, G, P + 3, D, fmt, dtype)
        vals = _fill(prefix, 0, P, 5000, 2.0)
    wide = _rand((B * T, H * D + 16), dtype, 99).cuda()
    q = wide[:, 8:8 + H * D]
    out_wide = torch.full((B * T, H * D + 8), 3.0, dtype=dtype).cuda()
    attn = KVAttention(cache, heads=H, tokens=T, prefix=prefix, prefix_len=P, causal=causal, scale=0.11)
    if attn.workspace is not None:
        attn.workspace[4096:].fill_(0xFF)                                          # NaN: only the counters need initialisation
    out = attn(q, torch.tensor(lens, dtype=torch.int32).cuda(), out=out_wide[:, :H * D])
    torch.cuda.synchronize()
    assert (out_wide[:, H * D:] == 3.0).all()
    _check(out, q, per_slot, vals, H, G, T, 0.11, causal, f"{fmt} {dtype}")
    # the same bits again, and with a host-side length where all slots have one
    assert torch.equal(attn(q, torch.tensor(lens, dtype=torch.int32).cuda()), out)
    n = max(lens)
    a = attn(q, torch.full((B,), n, dtype=torch.int32).cuda()) if T <= n else None
    if a is not None:
        assert torch.equal(torch.nan_to_num(a.float(), nan=9.0), torch.nan_to_num(attn(q, n).float(), nan=9.0))


@pytest.mark.parametrize("fmt", ["mx8", "16"])
@pytest.mark.parametrize("H,G,T,lens,P", [(4, 4, 1, [2500, 700], 0), (8, 1, 1, [4001], 0), (4, 4, 6, [1999, 33], 0), (2, 1, 1, [300, 7, 1], 3500),
                                          (2, 2, 200, [2600], 0), (4, 2, 150, [400, 155], 1700), (2, 2, 40, [900, 41, 600], 700)])
def test_attention_over_long_caches(fmt, H, G, T, lens, P):
    """Keys split over workgroups and joined, for host hints from far too small to the capacity."""
    D, B, rows = 128, len(lens), max(lens) + 40
    cache = _poisoned(B, G, rows, D, fmt, BF)
    per_slot = [_fill(cache, b, n, 100 * b + 1) for b, n in enumerate(lens)]
    prefix, vals = None, None
    if P:
        prefix = _poisoned(1, G, P, D, fmt, BF)
        vals = _fill(prefix, 0, P, 5000)
    q = _rand((B * T, H * D), BF, 98, 2.0).cuda()
    for kv_max in (0, 1, max(lens)):
        attn = KVAttention(cache, heads=H, tokens=T, prefix=prefix, prefix_len=P, kv_max=kv_max)
        out = attn(q, torch.tensor(lens, dtype=torch.int32).cuda())
        _check(out, q, per_slot, vals, H, G, T, 1.0 / math.sqrt(D), True, f"{fmt} kv_max {kv_max}")


@pytest.mark.parametrize("fmt", ["mx8", "16"])
@pytest.mark.parametrize("T,P", [(4, 0), (12, 0), (20, 40), (50, 0), (150, 0)])
def test_rows_a_query_does_not_see_have_no_influence(fmt, T, P):
    """NaN in the last rows (16 bits: infinities too): the queries before them are as if the rows were not there, the ones that see them NaN."""
    H, G, D, n = 4, 2, 128, 170
    cache = _poisoned(1, G, 200, D, fmt, BF)
    k, v = _fill(cache, 0, n, 1)
    prefix, vals = None, None
    if P:
        prefix = _poisoned(1, G, P, D, fmt, BF)
        vals = _fill(prefix, 0, P, 77)
    bad = n - T // 2                                                               # first row with a value that is not finite
    for r in range(bad, n):
        if fmt == "mx8":
            cache.k[0, :, r, 3], cache.v[0, :, r, 5], cache.v[0, :, r, 70] = 0x7F, 0x7F, 0xFF
        else:
            cache.k[0, :, r, 3], cache.v[0, :, r, 5], cache.v[0, :, r, 70] = float("nan"), float("inf"), float("nan")
    q = _rand((T, H * D), BF, 5).cuda()
    out = KVAttention(cache, heads=H, tokens=T, prefix=prefix, prefix_len=P)(q, n).view(T, H, D).cpu()
    sees = n - T + torch.arange(T) >= bad
    assert torch.isnan(out[sees]).all()                                            # a NaN key makes the whole row NaN
    clean = int((~sees).sum())
    for h in range(H):
        g = h // (H // G)
        kk, vv = k[g, :bad], v[g, :bad]
        if P:
            kk, vv = torch.cat((vals[0][g], kk)), torch.cat((vals[1][g], vv))
        want, tol = R.attention(q.cpu().view(T, H, D)[:clean, h], (P, kk), vv, 1.0 / math.sqrt(D), True, clean)
        assert ((out[:clean, h].double() - want).abs() <= tol).all()


@pytest.mark.parametrize("T", [2, 40, 140])
def test_values_that_are_not_finite_reach_only_their_channels(T):
    """16-bit rows: an infinite value in one channel makes that channel infinite (or NaN with its opposite) for the queries that see it."""
    H, D, n = 2, 128, 160
    cache = _poisoned(1, H, 176, D, "16", BF)
    k, v = _fill(cache, 0, n, 3)
    cache.v[0, :, n - 1, 9] = float("inf")
    cache.v[0, :, 0, 17], cache.v[0, :, 1, 17] = float("inf"), float("-inf")
    v[:, n - 1, 9], v[:, :2, 17] = 0.0, 0.0
    q = _rand((T, H * D), BF, 5).cuda()
    out = KVAttention(cache, heads=H, tokens=T)(q, n).view(T, H, D).cpu()
    assert torch.isnan(out[:, :, 17]).all() and (out[-1, :, 9] == float("inf")).all()
    rest = [d for d in range(D) if d not in (17, 9)]
    for h in range(H):
        want, tol = R.attention(q.cpu().view(T, H, D)[:, h], (0, k[h]), v[h], 1.0 / math.sqrt(D), True, T)
        off = (out[:, h].double() - want).abs()
        assert (off[:, rest] <= tol[:, rest]).all() and (off[:-1, 9] <= tol[:-1, 9]).all()


@pytest.mark.parametrize("gain", [30.0, 1e-3])
def test_peaked_and_flat_scores(gain):
    """Scores in the thousands (one key takes all) and near zero (every key alike)."""
    H, D, lens = 2, 128, [100, 190]
    for fmt in ("mx8", "16"):
        cache = _poisoned(2, H, 200, D, fmt, BF)
        per_slot = [_fill(cache, b, n, 7 * b + 1, gain) for b, n in enumerate(lens)]
        for T in (1, 20, 90):
            q = _rand((2 * T, H * D), BF, 6, gain).cuda()
            out = KVAttention(cache, heads=H, tokens=T, scale=0.25)(q, torch.tensor(lens, dtype=torch.int32).cuda())
            _check(out, q, per_slot, None, H, H, T, 0.25, True, f"{fmt} T {T}")


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("T", [1, 20, 100, 300])
def test_many_small_probabilities_count(dtype, T):
    """One key ahead of 1500 others whose probabilities, 2^-15.5 and less each, are fp16's subnormal numbers and together a part of the sum."""
    H, D, n = 1, 128, 1800
    cache = _poisoned(1, H, n, D, "16", dtype)
    k = torch.zeros(H, n, D)
    k[:, :, 0] = -1.0 - torch.arange(n) % 7 / 64.0
    k[:, 5, 0] = 0.0
    v = torch.ones(H, n, D)
    v[:, 5] = 0.0
    cache.k[0], cache.v[0] = k.to(dtype).cuda(), v.to(dtype).cuda()
    q = torch.zeros(T, H * D)
    q[:, 0] = 10.75                                                                # exp(-10.75) = 2^-15.51
    q = q.to(dtype).cuda()
    out = KVAttention(cache, heads=H, tokens=T, scale=1.0)(q, n)
    _check(out, q, [(k.to(dtype).double(), v.to(dtype).double())], None, H, H, T, 1.0, True)


def test_lengths_beyond_the_cache_are_clamped():
    H, D = 2, 128
    cache = _poisoned(2, H, 70, D, "mx8", BF)
    per_slot = [_fill(cache, b, 70, 7 * b + 1) for b in range(2)]
    for T in (1, 3, 66):
        q = _rand((2 * T, H * D), BF, 6).cuda()
        out = KVAttention(cache, heads=H, tokens=T)(q, torch.tensor([2 ** 31 - 1, 71], dtype=torch.int32).cuda())
        _check(out, q, per_slot, None, H, H, T, 1.0 / math.sqrt(D), True)
        assert (KVAttention(cache, heads=H, tokens=T)(q, torch.tensor([-5, -2 ** 31], dtype=torch.int32).cuda()) == 0).all()


@pytest.mark.parametrize("fmt", ["mx8", "16"])
def test_offsets_beyond_32_bits(fmt):
    """The last slot of a cache of more than 2^32 elements: written, read back and attended to."""
    H, D, rows, slots = 2, 128, 1 << 20, 17                                        # 17 * 2 * 2^20 * 128 = 4.56e9 elements each
    dt = torch.uint8 if fmt == "mx8" else BF
    k, v = (torch.empty(slots, H, rows, D, dtype=dt, device="cuda") for _ in range(2))
    ks, vs = (torch.empty(slots, H, rows, D // 32, dtype=torch.uint8, device="cuda") if fmt == "mx8" else None for _ in range(2))
    cache = KVCache.wrap(k, v, ks, vs, dtype=BF)
    n = 45
    lens = torch.zeros(slots, dtype=torch.int32)
    lens[-1] = rows - n
    past = torch.full((slots,), -1, dtype=torch.int32)
    past[-1] = rows - n
    qkv = _rand((slots * n, 3 * H * D), BF, 3)
    cos, sin = _tables(64, D, BF)
    q = cache.append(qkv.cuda(), cos.cuda(), sin.cuda(), past.cuda(), heads=H)
    x = qkv.view(slots, n, 3 * H, D)[-1]
    rot = R.rope(x[:, :2 * H], cos[63].expand(n, 1, D), sin[63].expand(n, 1, D))
    want_k, want_v = rot[:, H:].transpose(0, 1), x[:, 2 * H:].transpose(0, 1)
    if fmt == "mx8":
        want_k, want_v = (R.mx_decode(*R.mx_encode(t, R.top(BF))) for t in (want_k, want_v))
        gk, gv = cache.read(rows - n, n)
        assert torch.equal(gk[-1].cpu().double(), want_k) and torch.equal(gv[-1].cpu().double(), want_v)
        gk, gv = cache.slot(slots - 1).read(rows - n, n)
        assert torch.equal(gk[0].cpu().double(), want_k) and torch.equal(gv[0].cpu().double(), want_v)
    else:
        assert torch.equal(cache.k[-1, :, rows - n:].cpu(), want_k) and torch.equal(cache.v[-1, :, rows - n:].cpu(), want_v)
    # attention over the last n rows only: the same memory as a cache of n rows per head
    tail = KVCache.wrap(k[-1:, :, rows - n:], v[-1:, :, rows - n:], None if ks is None else ks[-1:, :, rows - n:],
                        None if vs is None else vs[-1:, :, rows - n:], dtype=BF)
    last = q.view(slots, n, -1)[-1].contiguous()
    out = KVAttention(tail, heads=H, tokens=n)(last, n)
    _check(out, last, [(want_k.double(), want_v.double())], None, H, H, n, 1.0 / math.sqrt(D), True)
    lens[:] = 0
    lens[-1] = 3                                                                   # ... and the whole cache, its last slot alone in use
    cut = [t[:, :3] for t in (want_k.double(), want_v.double())]
    for dst, src in ((k, rows - n), (v, rows - n)):
        dst[-1, :, :3] = dst[-1, :, src:src + 3]
    if fmt == "mx8":
        for dst in (ks, vs):
            dst[-1, :, :3] = dst[-1, :, rows - n:rows - n + 3]
    one = q.view(slots, n, -1)[:, 0].contiguous()
    out = KVAttention(cache, heads=H, kv_max=8)(one, lens.cuda())
    assert (out[:-1] == 0).all()
    _check(out[-1:], one[-1:], [cut], None, H, H, 1, 1.0 / math.sqrt(D), True)


def test_transposed_layout_and_one_slot_views():
    """Heads outside, slots inside: strides come from the tensors."""
    G, B, D, lens = 2, 3, 64, [20, 9, 33]
    k, v = (torch.full((G, B, 40, D), 0x7F, dtype=torch.uint8).cuda() for _ in range(2))
    ks, vs = (torch.full((G, B, 40, D // 32), 9, dtype=torch.uint8).cuda() for _ in range(2))
    cache = KVCache.wrap(*(t.transpose(0, 1) for t in (k, v, ks, vs)), dtype=HF)
    per_slot = [_fill(cache, b, n, 7 * b + 1) for b, n in enumerate(lens)]
    for T in (1, 66):
        q = _rand((B * T, 4 * D), HF, 6).cuda()
        out = KVAttention(cache, heads=4, tokens=T, causal=False)(q, torch.tensor(lens, dtype=torch.int32).cuda())
        _check(out, q, per_slot, None, 4, G, T, 1.0 / math.sqrt(D), False)
    one = KVAttention(cache.slot(1), heads=4, tokens=5)(q[:5], 9)
    _check(one, q[:5], per_slot[1:2], None, 4, G, 5, 1.0 / math.sqrt(D), True)


def test_odd_rows_of_64_values_and_slot_views():
    """33 rows of 64: scale rows of two bytes at every second address, slots alone as caches of their own, all written, read and attended to."""
    B, G, D, rows = 3, 1, 64, 33
    cache = _poisoned(B, G, rows, D, "mx8", BF)
    per_slot = [_fill(cache, b, rows, 7 * b + 1) for b in range(B)]
    for b in range(B):
        one = cache.slot(b)
        k, v = one.read(0, rows)
        assert torch.equal(k[0].cpu().double(), per_slot[b][0]) and torch.equal(v[0].cpu().double(), per_slot[b][1])
        for T in (1, 30, 33):
            q = _rand((T, 2 * D), BF, 6).cuda()
            _check(KVAttention(one, heads=2, tokens=T)(q, rows), q, per_slot[b:b + 1], None, 2, G, T, 1.0 / math.sqrt(D), True)
    x = _rand((1, 4 * D), BF, 8)
    cos, sin = (t.cuda() for t in _tables(64, D, BF))
    cache.slot(1).append(x.cuda(), cos, sin, 32, heads=2)
    code, byte = R.mx_encode(x.view(4, D)[3], R.top(BF))
    assert torch.equal(cache.v[1, 0, 32].cpu(), code) and torch.equal(cache.v_scale[1, 0, 32].cpu(), byte)
    k, v = cache.read(0, 0)
    assert k.shape == (B, G, 0, D) and v.shape == k.shape


def test_lengths_plus_the_new_rows():
    """plus = T on the lengths before the append: the same bits as lengths that count the new rows; idle slots stay idle."""
    H, D = 2, 128
    cache = _poisoned(3, H, 80, D, "mx8", BF)
    for b in range(3):
        _fill(cache, b, 80, 7 * b + 1)
    for T in (1, 4, 70):
        q = _rand((3 * T, H * D), BF, 6).cuda()
        attn = KVAttention(cache, heads=H, tokens=T)
        a = attn(q, torch.tensor([5, -1, 80 - T], dtype=torch.int32).cuda(), plus=T)
        b = attn(q, torch.tensor([5 + T, 0, 80], dtype=torch.int32).cuda())
        assert torch.equal(a, b) and (a.view(3, T, -1)[1] == 0).all()


# ------------------------------------------------------------------------------------------------ streams, graphs, the operators together
def test_a_captured_step_replays_with_new_lengths():
    """append + attention of one token in a graph whose lengths live on the device, replayed between eager work; a second captured object
    with a workspace of its own; both against the eager calls."""
    H, G, D, B, rows, P = 4, 2, 128, 3, 600, 300
    cos, sin = (t.cuda() for t in _tables(1024, D, BF))
    prefix = _poisoned(1, G, P, D, "mx8", BF)
    _fill(prefix, 0, P, 50)

    def fresh():
        c = _poisoned(B, G, rows, D, "mx8", BF)
        for b in range(B):
            _fill(c, b, 400 + b, 9 * b)
        return c
    cache, twin = fresh(), fresh()
    past = torch.tensor([400, 401, 402], dtype=torch.int32).cuda()
    qkv = torch.zeros(B, (H + 2 * G) * D, dtype=BF).cuda()
    attns = [KVAttention(cache, heads=H, prefix=prefix, prefix_len=P), KVAttention(cache, heads=H)]
    outs = [torch.empty(B, H * D, dtype=BF).cuda() for _ in range(2)]
    q_buf, n_buf = torch.empty(B, H * D, dtype=BF).cuda(), torch.empty(B, dtype=torch.int32).cuda()

    def step():
        cache.append(qkv, cos, sin, past, heads=H, pos_base=P, q_out=q_buf)
        torch.add(past, 1, out=n_buf)
        for a, o in zip(attns, outs):
            a(q_buf, n_buf, out=o)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    ref = [KVAttention(twin, heads=H, prefix=prefix, prefix_len=P), KVAttention(twin, heads=H)]
    for i in range(5):
        qkv.copy_(_rand(qkv.shape, BF, 60 + i).cuda())
        graph.replay()
        want_q = twin.append(qkv, cos, sin, past, heads=H, pos_base=P)
        want = [a(want_q, past + 1) for a in ref]
        torch.cuda.synchronize()
        assert torch.equal(q_buf, want_q)
        for o, w in zip(outs, want):
            assert torch.equal(o, w)
        past += 1


def test_calls_on_another_stream_are_ordered_there():
    H, D, n = 2, 128, 1500
    cache = _poisoned(1, H, n, D, "mx8", BF)
    vals = _fill(cache, 0, n, 1)
    q = _rand((1, H * D), BF, 2).cuda()
    attn = KVAttention(cache, heads=H)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        q2 = q * 2
        out = attn(q2, n)
    side.synchronize()
    _check(out, q2, [vals], None, H, H, 1, 1.0 / math.sqrt(D), True)


@pytest.mark.parametrize("fmt,dtype", [("mx8", BF), ("16", HF)])
def test_a_conversation_through_all_of_them(fmt, dtype):
    """A prompt into a one-slot prefix cache (one chunk of 70 tokens, one of 9), then four slots behind it: a chunk of 5 tokens, single
    tokens, and a step with one slot idle - every output against attention over all rows written so far, and the rows read back."""
    H, G, D, B, rows = 4, 2, 128, 4, 64
    cos, sin = _tables(256, D, dtype)
    cd, sd = cos.cuda(), sin.cuda()
    scale = 1.0 / math.sqrt(D)

    def rows_of(x, pos):
        """What the cache holds for x [T, (H + 2G) D] at the positions."""
        x = x.view(-1, H + 2 * G, D)
        k = R.rope(x[:, H:H + G], cos[pos].unsqueeze(1), sin[pos].unsqueeze(1)).transpose(0, 1)
        v = x[:, H + G:].transpose(0, 1)
        return [R.mx_decode(*R.mx_encode(t, R.top(dtype))) if fmt == "mx8" else t.double() for t in (k, v)]
    prefix = KVCache.new(1, G, 96, D, fmt, dtype)
    own = [torch.zeros(G, 0, D, dtype=torch.float64) for _ in range(2)]
    P = 0
    for i, T in enumerate((70, 9)):
        x = _rand((T, (H + 2 * G) * D), dtype, i)
        q = prefix.append(x.cuda(), cd, sd, P, heads=H)
        out = KVAttention(prefix, heads=H, tokens=T)(q, P + T)
        own = [torch.cat((a, b), 1) for a, b in zip(own, rows_of(x, torch.arange(P, P + T)))]
        P += T
        _check(out, q, [own], None, H, G, T, scale, True, f"prompt chunk {i}")
    if fmt == "mx8":
        k, v = prefix.read(0, P)
        assert torch.equal(k[0].cpu().double(), own[0]) and torch.equal(v[0].cpu().double(), own[1])
    shared, slots = own, [[torch.zeros(G, 0, D, dtype=torch.float64) for _ in range(2)] for _ in range(B)]
    cache = _poisoned(B, G, rows, D, fmt, dtype)
    lens = [0] * B
    for i, T in enumerate((5, 1, 1, 3, 1)):
        active = [b for b in range(B) if not (i == 2 and b == 1)]
        x = _rand((B * T, (H + 2 * G) * D), dtype, 20 + i)
        past = torch.tensor([lens[b] if b in active else -1 for b in range(B)], dtype=torch.int32)
        q = cache.append(x.cuda(), cd, sd, past.cuda(), heads=H, pos_base=P)
        for b in active:
            new = rows_of(x.view(B, T, -1)[b], P + lens[b] + torch.arange(T))
            slots[b] = [torch.cat((a, n), 1) for a, n in zip(slots[b], new)]
            lens[b] += T
        now = torch.tensor([lens[b] if b in active else 0 for b in range(B)], dtype=torch.int32)
        out = KVAttention(cache, heads=H, tokens=T, prefix=prefix, prefix_len=P)(q, now.cuda())
        seen = [slots[b] if b in active else [t[:, :0] for t in slots[b]] for b in range(B)]
        _check(out, q, seen, shared, H, G, T, scale, True, f"step {i}")


def test_python_calls_refuse_what_does_not_fit():
    c = KVCache.new(2, 2, 16, 128, "mx8", BF)
    cos, sin = (t.cuda() for t in _tables(16, 128, BF))
    qkv = torch.zeros(2, 6 * 128, dtype=BF).cuda()
    for bad in (qkv.float(), qkv[:, :-128], qkv.cpu(), qkv.t()):
        with pytest.raises(ValueError):
            c.append(bad, cos, sin, 0, heads=2)
    with pytest.raises(ValueError, match="int32"):
        c.append(qkv, cos, sin, torch.zeros(2, dtype=torch.int64).cuda(), heads=2)
    with pytest.raises(ValueError, match="cos / sin"):
        c.append(qkv, cos.float(), sin, 0, heads=2)
    with pytest.raises(ValueError, match="divide"):
        c.append(torch.zeros(3, 6 * 128, dtype=BF).cuda(), cos, sin, 0, heads=2)
    with pytest.raises(L.SeedmiError):
        c.append(qkv, cos, sin, 16, heads=2)
    with pytest.raises(L.SeedmiError):
        c.read(9, 8)
    a = KVAttention(c, heads=2)
    q = torch.zeros(2, 256, dtype=BF).cuda()
    for bad in (q[:1], q.half(), q[:, :128]):
        with pytest.raises(ValueError):
            a(bad, 4)
    with pytest.raises(L.SeedmiError):
        a(q, 17)
    with pytest.raises(ValueError):
        KVAttention(c, heads=3)
    with pytest.raises(IndexError):
        c.slot(2)
