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
