#!/usr/bin/env python
"""Times of the KV caches by handle beside their floors, plain forms and the static 16-bit cache (seed_amd/kv_cache.py, LlamaEngine.forward_kv).

    python tools/kv_bench.py rates               copy and product rates of the card, for the floors
    python tools/kv_bench.py cases [NAME,..]     perf/operators.py's listed cases, plain form and kernels in turn
    python tools/kv_bench.py run [NAME,..]       20 passes of the kernels of each case, for a kernel trace
    python tools/kv_bench.py more                shapes without a listed case, each with its floor
    python tools/kv_bench.py static              attention beside the static cache's kernel
    python tools/kv_bench.py steps               8B greedy steps at B = 32: static cache, 16-bit and 8-bit handles
    python tools/kv_bench.py logits              what 8-bit rows do to a model's logits (8B, synthetic weights; the static path's rounding as a yardstick)

Times are microseconds of a call among others, host call included: the median of seven rounds of calls that take turns over two or three sets of
inputs.  Floors: bytes at COPY, operations at PRODUCT, whichever takes longer."""
import math
import os
import statistics
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import perf.operators as P  # noqa: E402
from seed_amd import config as C  # noqa: E402
from seed_amd import lib as L  # noqa: E402
from seed_amd.kv_cache import KVAttention, KVCache, LayerCaches  # noqa: E402

COPY, PRODUCT = 5.1e12, 1.284e15                                                   # bytes/s, flop/s: `rates` on this card
BF, HF = torch.bfloat16, torch.float16


def us(calls, n=0, rounds=7):
    """Microseconds a call; ``calls`` take turns.  n = 0: as many as take some 5 ms, 20 at least."""
    for f in calls:
        f()
    if not n:
        n = max(20, min(300, int(5000 / us(calls, 10, 3))))
    times = []
    for _ in range(rounds):
        torch.cuda.synchronize()
        t = time.perf_counter()
        for i in range(n):
            calls[i % len(calls)]()
        torch.cuda.synchronize()
        times.append((time.perf_counter() - t) / n * 1e6)
    return statistics.median(times)


def floor(nbytes, flops=0):
    return max(nbytes / COPY, flops / PRODUCT) * 1e6


def rates():
    x = torch.empty(1 << 30, dtype=torch.uint8, device="cuda")
    y = torch.empty_like(x)
    a, b = (torch.randn(8192, 8192, device="cuda", dtype=BF) for _ in range(2))
    print(f"copy of a gigabyte {2 * x.numel() / us([lambda: y.copy_(x)]) / 1e6:.2f} TB/s (read + write)")
    print(f"8192^3 product, bf16 {2 * 8192 ** 3 / us([lambda: torch.mm(a, b)]) / 1e6:.0f} TFLOP/s", flush=True)


def _wanted(names):
    return [c for c in P.listed() if not names or c["name"] in names]


def cases(names):
    ratios = []
    for c in _wanted(names):
        w = P.work(c)
        P.own = False
        plain = [P.prepare(c, s) for s in range(2)]
        a = us([lambda s=s: P.run(s) for s in plain], n=6 if w["flops"] > 1e11 else 20, rounds=3)
        del plain
        P.own = True
        own = [P.prepare(c, s) for s in range(3)]
        b = us([lambda s=s: P.run(s) for s in own])
        del own
        ratios.append(a / b)
        print(f"{c['name']:20s} {w['bytes'] / 1e6:8.2f} MB {w['flops'] / 1e9:7.2f} GF  floor {floor(w['bytes'], w['flops']):7.2f}  plain {a:8.1f}  kernels {b:7.2f}  "
              f"({w['bytes'] / b / 1e6:.2f} TB/s, {w['flops'] / b / 1e6:.0f} TFLOP/s)", flush=True)
    print(f"geometric mean of plain / kernels over {len(ratios)} cases: {math.exp(statistics.mean(map(math.log, ratios))):.1f}")


def run(names):
    P.own = True
    for c in _wanted(names):
        sets = [P.prepare(c, s) for s in range(3)]
        torch.cuda.synchronize()
        for i in range(20):
            P.run(sets[i % 3])
        torch.cuda.synchronize()
        print(c["name"], flush=True)


def _cache(B, G, rows, D, fmt, dtype):
    c = KVCache.new(B, G, rows, D, fmt, dtype)
    for x in (c.k, c.v):
        x.random_(0, 100) if fmt == "mx8" else x.normal_()
    if fmt == "mx8":
        c.k_scale.fill_(122)
        c.v_scale.fill_(122)
    return c


def _attend(B, H, G, T, past, fmt, dtype=BF, D=128, prefix=0):
    n = past + T
    sets = []
    for _ in range(2):
        c, shared = _cache(B, G, n, D, fmt, dtype), _cache(1, G, prefix, D, fmt, dtype) if prefix else None
        q = torch.randn(B * T, H * D, device="cuda").to(dtype)
        sets.append((KVAttention(c, heads=H, tokens=T, kv_max=n, prefix=shared, prefix_len=prefix), q, torch.empty_like(q)))
    t = us([lambda s=s: s[0](s[1], n, out=s[2]) for s in sets])
    row = 2 * G * (D + D // 32 if fmt == "mx8" else 2 * D)
    nbytes = 4 * B * T * H * D + row * (B * n + prefix)
    flops = 4 * H * D * B * (T * n - T * (T - 1) // 2 + T * prefix)
    return t, floor(nbytes, flops), nbytes, flops


def more():
    for dtype in (BF, HF):
        for B, T in ((32, 1), (8, 649)):
            H, D, rows = 40, 128, 700
            cs = [_cache(B, H, rows, D, "16", dtype) for _ in range(2)]
            qkv = torch.randn(B * T, 3 * H * D, device="cuda").to(dtype)
            cos, sin = (torch.rand(rows, D, device="cuda").to(dtype) for _ in range(2))
            out = torch.empty(B * T, H * D, dtype=dtype, device="cuda")
            t = us([lambda c=c: c.append(qkv, cos, sin, 0, heads=H, q_out=out) for c in cs])
            print(f"append 16-bit rows {str(dtype)[6:]:8s} {B} x {T} x {H} heads: floor {floor(12 * B * T * H * D):6.1f}  {t:6.1f} us", flush=True)
    shapes = [("prompt from empty", 8, 40, 40, 649, 0, 128, 0), ("prompt from empty", 1, 32, 32, 649, 0, 128, 0), ("an image behind a turn", 8, 40, 40, 34, 600, 128, 0),
              ("100 rows behind 549", 8, 40, 40, 100, 549, 128, 0), ("17 rows behind 600", 8, 40, 40, 17, 600, 128, 0), ("second chunk", 2, 32, 32, 2048, 1953, 128, 0),
              ("one token", 32, 32, 32, 1, 4095, 128, 0), ("one token", 32, 32, 32, 1, 2047, 64, 0), ("second chunk", 2, 32, 32, 2048, 1953, 64, 0), ("100 rows behind 549", 8, 40, 40, 100, 549, 64, 0),
              ("prefix, 4 tokens", 16, 32, 32, 4, 0, 128, 2000), ("prefix, 60 tokens", 4, 40, 40, 60, 0, 128, 649), ("prefix, 1024 tokens", 2, 32, 32, 1024, 0, 128, 1000)]
    for name, B, H, G, T, past, D, prefix in shapes:
        for fmt, dtype in (("mx8", BF), ("16", BF), ("mx8", HF)):
            t, fl, nbytes, flops = _attend(B, H, G, T, past, fmt, dtype, D, prefix)
            print(f"{name:22s} {fmt:3s} {str(dtype)[6:]:8s} B {B} H {H}:{G} T {T} past {past} prefix {prefix} head_dim {D}: floor {fl:6.1f}  {t:6.1f} us  "
                  f"({nbytes / t / 1e6:.2f} TB/s, {flops / t / 1e6:.0f} TFLOP/s)", flush=True)


def static():
    lib = L.load()
    D = 128
    for B, H, T, past in ((8, 40, 649, 0), (2, 32, 2048, 1953), (8, 40, 17, 600), (32, 32, 1, 1023)):
        n = past + T
        sets = [(torch.randn(B, H, n, D, device="cuda", dtype=BF), torch.randn(B, H, n, D, device="cuda", dtype=BF)) for _ in range(2)]
        q = torch.randn(B * T, H * D, device="cuda", dtype=BF)
        out = torch.empty_like(q)
        a = us([lambda k=k, v=v: L.check(lib.seedmi_llama_attention_bf16(L.ptr(q), H * D, L.ptr(k), L.ptr(v), L.ptr(out), H * D, B, T, H, D, n, past,
                                                                         1 / math.sqrt(D), 0, None, L.stream_ptr()), "static", lib) for k, v in sets])
        del sets
        b, c = (_attend(B, H, H, T, past, fmt)[0] for fmt in ("16", "mx8"))
        print(f"{B} x {H} heads, {T} new behind {past}: static {a:.1f}  16-bit handle {b:.1f}  8-bit handle {c:.1f} us", flush=True)


def _engine_8b(B, tmax, successor=False):
    from seed_amd.llama_engine import LlamaEngine
    from seed_amd.weights import make_llama_state_dict, make_llama_successor_state_dict
    cfg = C.LLAMA_8B
    sd = make_llama_successor_state_dict(cfg, device="cuda", dtype=BF)[0] if successor else make_llama_state_dict(cfg, device="cuda", dtype=BF)
    return cfg, LlamaEngine(sd, cfg, batch_cap=B, tmax=tmax)


def steps():
    B = 32
    cfg, eng = _engine_8b(B, 2048)
    for c in eng.k_cache + eng.v_cache:
        c.normal_()
    tok = torch.ones(B, 1, dtype=torch.int64, device="cuda")
    for past in (100, 1000, 1900):
        eng.past_len = past
        replay, _ = eng.capture_decode_graph(tok, 2040 - past)
        line = f"8B greedy step, B = {B}, behind {past} rows: static 16-bit {us([lambda: replay(1)], 8) / 1e3:.3f} ms"
        for fmt in ("16", "mx8"):
            kv = LayerCaches(_cache(B, cfg.heads, 2048, cfg.head_dim, fmt, BF) for _ in range(cfg.layers))
            lens = torch.full((B,), past, dtype=torch.int32, device="cuda")
            step = lambda: eng.forward_kv(tok, kv, lens, past + 40, last_only=True)  # noqa: E731
            step()
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step()
            line += f"  handle {fmt} {us([graph.replay], 8) / 1e3:.3f} ms"
            del kv, graph
        print(line, flush=True)


def logits():
    B, T, n = 4, 500, 20
    for successor in (False, True):
        cfg, eng = _engine_8b(B, T + n, successor)
        ids = torch.randint(3, cfg.vocab, (B, T + n), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
        cuts = [(0, T)] + [(T + i, 1) for i in range(n)]
        out = {"static": [eng.forward(ids[:, a:a + m], past_len=a).double() for a, m in cuts]}
        for fmt in ("16", "mx8"):
            kv = eng.new_kv(B, T + n, fmt)
            out[fmt] = [eng.forward_kv(ids[:, a:a + m], kv, torch.full((B,), a, dtype=torch.int32, device="cuda"), a).double() for a, m in cuts]
            del kv
        for name, part in (("prompt of 500", slice(0, 1)), ("20 steps behind it", slice(1, None))):
            ref, line = torch.cat(out["16"][part], 1), f"{'peaked' if successor else 'random'} weights, {name}, against 16-bit handles:"
            for other in ("static", "mx8"):
                x = torch.cat(out[other][part], 1)
                line += (f"  {other}: relative difference {((x - ref).norm() / ref.norm()).item():.4f}, same best token "
                         f"{(x.argmax(-1) == ref.argmax(-1)).double().mean().item():.3f}")
            print(line, flush=True)
        del eng, out


if __name__ == "__main__":
    what, names = (sys.argv + ["rates"])[1], set(sys.argv[2].split(",")) if len(sys.argv) > 2 else set()
    {"rates": rates, "cases": lambda: cases(names), "run": lambda: run(names), "more": more, "static": static, "steps": steps, "logits": logits}[what]()
