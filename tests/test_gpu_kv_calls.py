"""KV caches by handle on the GPU: calls around captures and streams, and values at the edges of the types."""
import math

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
