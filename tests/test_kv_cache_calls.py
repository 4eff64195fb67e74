"""KV caches by handle, without a GPU: which host-side calls are taken, which are refused, and that a refused call leaves nothing behind."""
import contextlib
import ctypes as C
import os
import subprocess
import sys
import types

import pytest
import torch

from seed_amd import config as CFG
from seed_amd import kv_cache
from seed_amd import lib as L
from seed_amd.kv_cache import KVAttention, KVCache, LayerCaches
from seed_amd.llama_engine import LlamaEngine

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


# ------------------------------------------------------------------------------------------------ rows of a call
@pytest.mark.parametrize("rows,tokens", [(8, 3), (10, 4), (12, 5), (7, 8), (4, 0), (4, -2)])
def test_rows_that_tokens_do_not_divide_are_refused(rows, tokens):
    """tokens=3 asks for slots of three rows: eight rows are not two slots of four."""
    with pytest.raises(ValueError, match="do not divide"):
        KVCache._batch(types.SimpleNamespace(slots=8), "append", rows, 0, tokens)


@pytest.mark.parametrize("rows,tokens,lens,want", [(8, 4, 0, (2, 4)), (8, 1, 0, (8, 1)), (3, 3, 0, (1, 3)), (8, None, 0, (4, 2)),
                                                   (6, None, torch.zeros(3, dtype=torch.int32), (3, 2)), (6, 2, torch.zeros(4, dtype=torch.int32), (3, 2))])
def test_slots_and_tokens_of_a_call(rows, tokens, lens, want):
    assert KVCache._batch(types.SimpleNamespace(slots=8 if tokens else 4), "append", rows, lens, tokens) == want


# ------------------------------------------------------------------------------------------------ workspaces and captures
class _Called(Exception):
    """A stub's method that must not be reached was."""


def _on_the_host(slots=2, heads=2, rows=4096, dim=128):
    """A 16-bit cache whose tensors are on the CPU, for what the Python side decides by itself (no call of it may launch)."""
    c = KVCache.__new__(KVCache)
    c.k = c.v = torch.zeros(slots, heads, rows, dim, dtype=torch.bfloat16)
    c.k_scale = c.v_scale = None
    c.dtype, c.device, c.format, c.index = torch.bfloat16, torch.device("cpu"), "16", -1
    c.slots, c.kv_heads, c.rows, c.head_dim = slots, heads, rows, dim
    c.lib = L.load()
    c.struct = L.KVCacheStruct(c.k.data_ptr(), c.v.data_ptr(), 0, 0, heads * rows, rows, slots, rows, heads, dim, L.KV_16BIT)
    c._ref = C.byref(c.struct)
    c._append, c._read = c.lib.seedmi_kv_append, c.lib.seedmi_kv_read
    return c


def test_an_attention_with_a_workspace_is_not_made_during_a_capture(monkeypatch):
    """The initialisation of the arrival counters would be recorded and not run: calls before the first replay would count on whatever the
    allocation held, and their rows stay unwritten."""
    def reached(*a, **k):
        raise _Called
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    monkeypatch.setattr(kv_cache, "_call", reached)
    cache = _on_the_host()
    assert cache.lib.seedmi_kv_attention_workspace_bytes(cache._ref, 2, 1, 2, 0, 0) > 0
    with pytest.raises(L.SeedmiError, match="before the capture"):
        KVAttention(cache, heads=2)


def _engine_on_the_host(ws, kv_ws, monkeypatch):
    """A LlamaEngine without weights on the CPU, as forward_kv sees it up to its first library call."""
    e = LlamaEngine.__new__(LlamaEngine)
    e.cfg, e.dtype, e.device, e.lib = CFG.LLAMA_TINY, torch.bfloat16, torch.device("cpu"), L.load()
    e.w = L.LlamaWeights()
    e.w.hidden, e.w.layers, e.w.heads, e.w.ffn, e.w.vocab = e.cfg.hidden, e.cfg.layers, e.cfg.heads, e.cfg.ffn, e.cfg.vocab
    e.vocab_pad, e.w.vocab_pad, e.w.max_pos = e.cfg.vocab, e.cfg.vocab, e.cfg.max_pos
    e._ws, e._ws_key, e._kv_ws, e._kv_captured = ws, (0, 0), kv_ws, []

    def reached(*a, **k):
        raise _Called
    monkeypatch.setattr(LlamaEngine, "new_workspace", reached)
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    return e


@pytest.mark.parametrize("missing", ["attention", "activations"])
def test_forward_kv_does_not_grow_its_workspaces_during_a_capture(monkeypatch, missing):
    """A warm-up with a smaller past_max than the captured call's: the larger workspace's counters would be initialised by the replays only."""
    cfg = CFG.LLAMA_TINY
    kv = LayerCaches([_on_the_host(2, cfg.heads, 4096, cfg.head_dim) for _ in range(cfg.layers)])
    need = L.load().seedmi_kv_attention_workspace_bytes(kv.array, 2, 1, cfg.heads, 4000, 0)
    assert need > 0
    big = torch.zeros(1 << 24, dtype=torch.uint8)
    e = _engine_on_the_host(big if missing == "attention" else big[:1], big[:need - 1] if missing == "attention" else big, monkeypatch)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(L.SeedmiError, match="once before the capture"):
        e.forward_kv(torch.zeros(2, 1, dtype=torch.int64), kv, torch.zeros(2, dtype=torch.int32), 3999)


# ------------------------------------------------------------------------------------------------ numbers beyond 32 bits
BIG = 1 << 32


def test_numbers_beyond_32_bits_are_refused(monkeypatch):
    """ctypes passes the low 32 bits of an int: 2^32 + 5 rows would be 5."""
    def reached(*a, **k):
        raise _Called
    monkeypatch.setattr(kv_cache, "_call", reached)
    monkeypatch.setattr(kv_cache, "_current_stream", lambda index: 0)
    c = _on_the_host(rows=64)
    q, qkv = torch.zeros(2, 256, dtype=torch.bfloat16), torch.zeros(2, 768, dtype=torch.bfloat16)
    cos = torch.zeros(64, 128, dtype=torch.bfloat16)
    attn = KVAttention(c, heads=2)
    assert attn.workspace is None
    ok = [lambda: c.append(qkv, cos, cos, 5, heads=2), lambda: c.read(5, 2), lambda: attn(q, 5), lambda: attn(q, 5, plus=1)]
    for call in ok:
        with pytest.raises(_Called):
            call()
    bad = [lambda: c.append(qkv, cos, cos, BIG + 5, heads=2), lambda: c.append(qkv, cos, cos, 5, heads=2, pos_base=BIG), lambda: c.read(BIG, 2),
           lambda: c.read(5, BIG), lambda: attn(q, BIG + 5), lambda: attn(q, 5, plus=BIG), lambda: attn(q, (1 << 31) - 1, plus=1),
           lambda: KVAttention(c, heads=2, kv_max=BIG + 5), lambda: KVAttention(c, heads=2, tokens=BIG + 1),
           lambda: KVAttention(c, heads=BIG + 2), lambda: KVAttention(c, heads=2, prefix=c, prefix_len=BIG + 1)]
    for call in bad:
        with pytest.raises(ValueError, match="beyond 32 bits"):
            call()


@pytest.mark.parametrize("kw", [dict(past_max=BIG + 5), dict(past_max=-BIG), dict(past_max=5, prefix_len=BIG + 1)])
def test_forward_kv_refuses_numbers_beyond_32_bits(monkeypatch, kw):
    cfg = CFG.LLAMA_TINY
    kv = LayerCaches([_on_the_host(2, cfg.heads, 64, cfg.head_dim) for _ in range(cfg.layers)])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    e = _engine_on_the_host(None, None, monkeypatch)
    with pytest.raises(ValueError, match="beyond 32 bits"):
        e.forward_kv(torch.zeros(2, 1, dtype=torch.int64), kv, torch.zeros(2, dtype=torch.int32), prefix=kv if "prefix_len" in kw else None, **kw)
    with pytest.raises(_Called):
        e.forward_kv(torch.zeros(2, 1, dtype=torch.int64), kv, torch.zeros(2, dtype=torch.int32), 5)


# ------------------------------------------------------------------------------------------------ the forward at the C ABI
FAKE = 0x10000                                            # aligned, never dereferenced on these paths


def _handle(**kw):
    h = L.KVCacheStruct(FAKE, FAKE, FAKE, FAKE, 2 * 64, 64, 4, 64, 2, 128, L.KV_MX8)
    for k, v in kw.items():
        setattr(h, k, v)
    return h


@pytest.mark.parametrize("model,cache", [(dict(heads=0), {}), (dict(heads=0), dict(kv_heads=0)), (dict(heads=-2), dict(kv_heads=-2)),
                                         (dict(hidden=0), {}), (dict(hidden=255), {}), (dict(layers=0), {}), (dict(layers=-1), {})])
def test_a_model_without_heads_or_layers_is_refused(model, cache):
    """An error code, not a division by zero, from a process of its own."""
    code = f"""
import ctypes as C
from seed_amd import lib as L
w = L.LlamaWeights()
for k, v in dict(dict(hidden=256, layers=1, heads=2, max_pos=64), **{model}).items():
    setattr(w, k, v)
h = L.KVCacheStruct({FAKE}, {FAKE}, {FAKE}, {FAKE}, 128, 64, 4, 64, 2, 128, L.KV_MX8)
for k, v in {cache}.items():
    setattr(h, k, v)
kv = (L.KVCacheStruct * 1)(h)
print(L.load().seedmi_llama_forward_kv(C.byref(w), kv, None, 0, {FAKE}, 4, 2, {FAKE}, 8, 0, {FAKE}, 64, None, 0, {FAKE}, 0, None))
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=ROOT)
    assert r.returncode == 0 and r.stdout.split()[-1] == "-1", (r.returncode, r.stderr)


def _forward_kv(kv, prefix=None, **kw):
    w = L.LlamaWeights()
    w.hidden, w.layers, w.heads, w.ffn, w.vocab, w.vocab_pad, w.max_pos, w.tmax, w.batch_cap = 256, 2, 2, 512, 64, 64, 4096, 64, 4
    w.embed = w.cos_t = w.sin_t = FAKE
    layers = (L.LlamaLayer * 2)()
    w.layer = C.cast(layers, C.POINTER(L.LlamaLayer))
    a = dict(plen=0, ids=FAKE, B=4, T=2, past=FAKE, past_max=8, last=0, logits=FAKE, ldl=64, aws=None, ab=0, ws=FAKE, wb=1 << 30)
    a.update(kw)
    kv = (L.KVCacheStruct * 2)(*kv)
    prefix = None if prefix is None else (L.KVCacheStruct * 2)(*prefix)
    return L.load().seedmi_llama_forward_kv(C.byref(w), kv, prefix, *a.values(), None)


BAD_LAYERS = [(dict(format=2), -2), (dict(k=None), -1), (dict(v_scale=None), -1), (dict(v=FAKE + 8), -3), (dict(head_rows=63), -1)]


@pytest.mark.parametrize("bad,code", BAD_LAYERS)
def test_a_bad_cache_of_a_later_layer_is_refused_before_anything_runs(bad, code):
    """(Here every launch fails, without a GPU: what comes back is the refusal only if nothing was launched before it.)"""
    assert _forward_kv([_handle(), _handle(**bad)]) == code


@pytest.mark.parametrize("bad,code", BAD_LAYERS[:4] + [(dict(rows=31), -1), (dict(head_dim=64), -1), (dict(kv_heads=1), -1),
                                                       (dict(format=L.KV_16BIT, k_scale=None, v_scale=None), -1)])
def test_a_bad_prefix_of_a_later_layer_is_refused_before_anything_runs(bad, code):
    assert _forward_kv([_handle(), _handle()], [_handle(slots=1), _handle(slots=1, **bad)], plen=32, aws=FAKE, ab=1 << 20) == code


def test_a_short_attention_workspace_is_refused_before_anything_runs():
    kv = [_handle(rows=1 << 12, slot_rows=2 << 12, head_rows=1 << 12) for _ in range(2)]
    need = L.load().seedmi_kv_attention_workspace_bytes(C.byref(kv[0]), 1, 1, 2, 4001, 0)
    assert need > 0
    for ws, n in ((None, 0), (FAKE, need - 1), (FAKE + 128, need)):
        assert _forward_kv(kv, B=1, T=1, past_max=4000, aws=ws, ab=n) == -3


# ------------------------------------------------------------------------------------------------ scale
@pytest.mark.parametrize("scale", [0.0, -0.1, float("inf"), float("nan"), 3.3e38, 2.5e38])
def test_scales_that_are_not_finite_in_base_2_exponents_are_refused(scale):
    """2.5e38 log2 e is beyond fp32: every score would be infinite, or NaN where it is 0."""
    h = _handle()
    rc = L.load().seedmi_kv_attention(C.byref(h), None, 0, FAKE, 256, FAKE, 256, 4, 1, 2, 8, None, 0, scale, 1, None, 0, None)
    assert rc == -1 and "scale" in L.load().seedmi_last_error().decode()
