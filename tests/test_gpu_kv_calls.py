"""KV caches by handle on the GPU: calls around captures and streams, and values at the edges of the types."""
import gc
import math
import weakref

import pytest
import torch

pytestmark = pytest.mark.gpu

from seed_amd import config as C  # noqa: E402
from seed_amd import lib as L  # noqa: E402
from seed_amd.kv_cache import KVAttention, KVCache  # noqa: E402
from seed_amd.llama_engine import LlamaEngine  # noqa: E402
from seed_amd.weights import make_llama_state_dict  # noqa: E402
from tests import _kv_ref as R  # noqa: E402

BF, HF = torch.bfloat16, torch.float16
CFG = C.LLAMA_TINY


def _rand(shape, dtype, seed, gain=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * gain).to(dtype)


def _lens(*n):
    return torch.tensor(n, dtype=torch.int32).cuda()


@pytest.fixture
def engine():
    return LlamaEngine(make_llama_state_dict(CFG, seed=11, norm_jitter=0.1), CFG, device="cuda", batch_cap=4, tmax=128)


# ------------------------------------------------------------------------------------------------ captures and streams
def test_an_attention_made_during_a_capture_is_refused():
    cache = KVCache.new(1, 2, 3000, 128, "16", BF)
    cache.k[0], cache.v[0] = _rand((2, 3000, 128), BF, 1).cuda(), _rand((2, 3000, 128), BF, 2).cuda()
    q = _rand((1, 256), BF, 3).cuda()
    want = KVAttention(cache, heads=2)(q, 2500)
    torch.cuda.synchronize()
    with pytest.raises(L.SeedmiError, match="before the capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            q + 1
            KVAttention(cache, heads=2)
    attn, graph = KVAttention(cache, heads=2), torch.cuda.CUDAGraph()
    assert attn.workspace is not None and torch.equal(attn(q, 2500), want)
    with torch.cuda.graph(graph):
        out = attn(q, 2500)
    assert torch.equal(attn(q, 2500), want)                                        # eager between the capture and the first replay
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_forward_kv_is_captured_after_a_call_of_its_size(engine):
    """A warm-up behind few rows, a capture behind many: refused, and the eager calls go on as before; after a warm-up of that size it is
    taken, and an eager call between the capture and the first replay gives the same bits."""
    B = 2
    kv, twin = engine.new_kv(B, 250), engine.new_kv(B, 250)
    tok = torch.tensor([[5], [7]]).cuda()
    past = _lens(0, 0)
    small = engine.forward_kv(tok, kv, past, 0, last_only=True)
    torch.cuda.synchronize()
    with pytest.raises(L.SeedmiError, match="once before the capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            tok + 1
            engine.forward_kv(tok, kv, past, 240, last_only=True)
    assert torch.equal(engine.forward_kv(tok, kv, past, 0, last_only=True), small)
    want = engine.forward_kv(tok, twin, past, 240, last_only=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = engine.forward_kv(tok, kv, past, 240, last_only=True)
    assert torch.equal(engine.forward_kv(tok, kv, past, 240, last_only=True), want)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_forward_kv_keeps_only_the_workspaces_that_graphs_replay_on(engine):
    """Prompts that grow step by step: every outgrown workspace is released, but for those of a captured call, whose replays go on."""
    kv = engine.new_kv(2, 250)
    old = []
    for T in (3, 20, 60, 130, 200):
        engine.forward_kv(torch.ones(1, T, dtype=torch.int64).cuda(), kv, _lens(0), 40 if T < 200 else 0, last_only=True)
        old.append((weakref.ref(engine._ws), None if engine._kv_ws is None else weakref.ref(engine._kv_ws)))
    gc.collect()
    assert old[0][0]() is None and old[-1][0]() is engine._ws
    assert len({id(w()) for w, _ in old if w() is not None}) == 1 and len({id(k()) for _, k in old if k is not None and k() is not None}) <= 1
    small = LlamaEngine(make_llama_state_dict(CFG, seed=11, norm_jitter=0.1), CFG, device="cuda", batch_cap=4, tmax=128)
    tok, past = torch.tensor([[5]]).cuda(), _lens(9)
    step = lambda: small.forward_kv(tok, kv, past, 240, last_only=True)  # noqa: E731
    want = step()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = step()
    captured = [weakref.ref(small._ws), weakref.ref(small._kv_ws)]
    small.forward_kv(torch.ones(2, 200, dtype=torch.int64).cuda(), kv, _lens(-1, 0), 50, last_only=True)
    small.resize_cache(tmax=64)
    gc.collect()
    assert all(w() is not None for w in captured) and small._ws is None
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_new_workspaces_of_forward_kv_are_ready_for_any_stream(engine):
    """The call that allocates them returns after their initialisation has run, on a busy stream too; calls on two streams with an event
    between them give what one stream gives."""
    kv, twin = engine.new_kv(2, 250), engine.new_kv(2, 250)
    ids, tok = torch.arange(60).view(2, 30).cuda(), torch.tensor([[5], [7]]).cuda()
    a = torch.randn(4096, 4096, device="cuda", dtype=BF)
    b = a @ a
    none = _lens(0, 0)
    engine.forward_kv(tok, kv, none, 0)                                            # (the kernels are loaded; the next call's workspaces are larger)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(300):
            torch.mm(a, a, out=b)
        busy = torch.cuda.Event()
        busy.record()
        first = engine.forward_kv(ids, kv, none, 0)
        assert busy.query()
    torch.cuda.current_stream().wait_stream(side)
    second = engine.forward_kv(tok, kv, _lens(30, 30), 240)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        third = engine.forward_kv(tok, kv, _lens(31, 31), 240)
    torch.cuda.synchronize()
    for got, x, n, most in ((first, ids, 0, 0), (second, tok, 30, 240), (third, tok, 31, 240)):
        assert torch.equal(got, engine.forward_kv(x, twin, _lens(n, n), most))


@pytest.mark.parametrize("fold", [True, False])
def test_a_captured_step_replays_with_and_without_folded_norms(fold):
    """Without folded norms the step clears the split-K flags itself: replays with eager steps and synchronisations between them."""
    eng = LlamaEngine(make_llama_state_dict(CFG, seed=11, norm_jitter=0.1), CFG, device="cuda", batch_cap=4, tmax=128, fold_norm=fold)
    kv, twin = eng.new_kv(2, 250), eng.new_kv(2, 250)
    tok, past = torch.tensor([[5], [7]]).cuda(), _lens(0, 0)
    step = lambda c: eng.forward_kv(tok, c, past, 200, last_only=True)  # noqa: E731
    step(kv)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(kv)
    for i in range(6):
        tok.fill_(11 + i)
        graph.replay()
        want = step(twin)
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
        past += 1
    eng.decode_status(2)


# ------------------------------------------------------------------------------------------------ calls together, captured, at the largest sizes
def _filled(B, G, rows, D, fmt, dtype, seed):
    c = KVCache.new(B, G, rows, D, fmt, dtype)
    for i, (x, s) in enumerate(((c.k, c.k_scale), (c.v, c.v_scale))):
        v = _rand((B, G, rows, D), dtype, seed + i)
        if fmt == "16":
            x.copy_(v)
        else:
            code, byte = R.mx_encode(v, R.top(dtype))
            x.copy_(code)
            s.copy_(byte)
    return c


def test_two_objects_and_a_graph_over_one_cache_at_the_same_time():
    """Two streams and a replaying graph, an object each, 30 calls in flight: every output as it is alone."""
    H, G, D, B, P = 8, 2, 128, 3, 900
    cache, prefix = _filled(B, G, 2000, D, "mx8", BF, 1), _filled(1, G, P, D, "mx8", BF, 5)
    lens = _lens(2000, 700, 1)
    make = [lambda: KVAttention(cache, heads=H), lambda: KVAttention(cache, heads=H, prefix=prefix, prefix_len=P),
            lambda: KVAttention(cache, heads=H, tokens=20, prefix=prefix, prefix_len=P)]
    qs = [_rand((B * t, H * D), BF, 7 + t).cuda() for t in (1, 1, 20)]
    want = [m()(q, lens) for m, q in zip(make, qs)]
    attns = [m() for m in make]
    assert all(a.workspace is not None for a in attns)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = attns[2](qs[2], lens)
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = [[], []]
    torch.cuda.synchronize()
    for _ in range(30):
        for s, a, q, g in zip(streams, attns, qs, got):
            with torch.cuda.stream(s):
                g.append(a(q, lens))
        with torch.cuda.stream(streams[2]):
            graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want[2])
    for g, w in zip(got, want):
        assert all(torch.equal(x, w) for x in g)


@pytest.mark.parametrize("T,P", [(20, 0), (60, 700), (300, 0), (200, 900)])
def test_captured_chunks_replay_with_new_lengths(T, P):
    """append and attention of more than one token per slot, with parts that a launch of its own joins, replayed as the lengths grow."""
    H, G, D, B, rows = 4, 2, 128, 2, 1700
    cos, sin = (_rand((4096, D), BF, 3 + i).clamp(-1, 1).cuda() for i in range(2))
    prefix = _filled(1, G, P, D, "mx8", BF, 30) if P else None
    cache, twin = _filled(B, G, rows, D, "mx8", BF, 9), _filled(B, G, rows, D, "mx8", BF, 9)
    make = lambda c: KVAttention(c, heads=H, tokens=T, prefix=prefix, prefix_len=P)  # noqa: E731
    attn, other = make(cache), make(twin)
    past, qkv, q = _lens(500, 3), torch.zeros(B * T, (H + 2 * G) * D, dtype=BF).cuda(), torch.empty(B * T, H * D, dtype=BF).cuda()
    out = torch.empty_like(q)

    def step():
        cache.append(qkv, cos, sin, past, heads=H, pos_base=P, q_out=q)
        attn(q, past, plus=T, out=out)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(3):
        qkv.copy_(_rand(qkv.shape, BF, 60 + i).cuda())
        graph.replay()
        want = other(twin.append(qkv, cos, sin, past, heads=H, pos_base=P), past, plus=T)
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
        past += T


@pytest.mark.parametrize("fmt", ["16", "mx8"])
@pytest.mark.parametrize("T", [1, 20, 60, 100, 300])
def test_the_longest_cache(fmt, T):
    """2^22 rows, the most that a cache may have: queries that single out four keys far apart, 30 ahead of the others, which have e^-30 2^22 <
    5e-7 of the sum together.  Tolerance: output and probabilities half a step each, scores of 30 to 2^-17, sums of at most 2^16 terms in
    a row."""
    D, n = 128, 1 << 22
    at = torch.tensor([0, n // 2 + 3, n - 70, n - 1])
    dt = BF if fmt == "16" else torch.uint8
    k, v = (torch.zeros(1, 1, n, D, dtype=dt, device="cuda") for _ in range(2))
    ks, vs = (torch.full((1, 1, n, D // 32), 127, dtype=torch.uint8, device="cuda") if fmt == "mx8" else None for _ in range(2))
    key = torch.zeros(4, D)
    key[:, 0] = torch.tensor([30.0, 32.0, 30.0, 32.0])
    val = _rand((4, D), BF, 2)
    if fmt == "16":
        k[0, 0, at.cuda()], v[0, 0, at.cuda()] = key.to(BF).cuda(), val.cuda()
        vals = val.double()
    else:
        for x, s, y in ((k, ks, key.to(BF)), (v, vs, val)):
            code, byte = R.mx_encode(y, R.top(BF))
            x[0, 0, at.cuda()], s[0, 0, at.cuda()] = code.cuda(), byte.cuda()
        vals = R.mx_decode(*R.mx_encode(val, R.top(BF)))
    q = torch.zeros(T, D)
    q[:, 0] = 1.0
    cache = KVCache.wrap(k, v, ks, vs, dtype=BF)
    out = KVAttention(cache, heads=1, tokens=T, scale=1.0, causal=False)(q.to(BF).cuda(), n).cpu().double()
    w = torch.softmax(key[:, 0].double(), 0)
    want, u = w @ vals, 2.0 ** -8
    tol = 1.01 * u * want.abs() + (1.02 * u + 2.0 ** -15 + 2 * 65536 * 2.0 ** -24) * (w @ vals.abs()) + 5e-7
    assert ((out - want).abs() <= tol).all(), ((out - want).abs() - tol).max().item()


def test_read_of_values_alone_and_append_of_the_first_slots():
    """seedmi_kv_read with one output; append with tokens= on fewer slots than there are lengths."""
    H, D, dtype = 2, 128, BF
    cache = _filled(4, H, 40, D, "mx8", dtype, 3)
    both = cache.read(5, 7)
    for i in range(2):
        out = torch.zeros_like(both[0])
        p = [None, None]
        p[i] = out.data_ptr()
        L.check(cache.lib.seedmi_kv_read(cache._ref, p[0], p[1], 4, 7, 5, None, L.stream_ptr()), "read", cache.lib)
        assert torch.equal(out, both[i])
    before = cache.k.clone()
    cos, sin = (_rand((64, D), dtype, 4 + i).cuda() for i in range(2))
    cache.append(_rand((6, 3 * H * D), dtype, 8).cuda(), cos, sin, _lens(1, 30, 9, 9), heads=H, tokens=3)
    changed = (cache.k != before).any(-1).any(1).cpu()
    assert changed[0, 1:4].all() and changed[1, 30:33].all() and int(changed.sum()) == 6


@pytest.mark.parametrize("B", [40, 70])
def test_more_slots_than_the_static_cache_has(B, engine):
    """One step of 40 and of 70 slots (the engine's own cache has 4): each slot's logits as in a call of four."""
    kv = engine.new_kv(B, 20, "16")
    ids = torch.randint(3, CFG.vocab, (B, 6), generator=torch.Generator().manual_seed(4)).cuda()
    past = torch.zeros(B, dtype=torch.int32).cuda()
    engine.forward_kv(ids[:, :5].contiguous(), kv, past, 0)
    past += 5
    got = engine.forward_kv(ids[:, 5:].contiguous(), kv, past, 5, last_only=True)
    for b in range(0, B, 13):
        one = engine.new_kv(1, 20, "16")
        engine.forward_kv(ids[b:b + 1, :5].contiguous(), one, past[:1] * 0, 0)
        want = engine.forward_kv(ids[b:b + 1, 5:].contiguous(), one, past[:1], 5, last_only=True)
        d = (got[b].double() - want[0].double()).norm() / want[0].double().norm()
        assert d.item() < 2e-2, (b, d.item())
