"""KV caches by handle, without a GPU: what the entry points and the Python classes refuse, the handle's layout, and the 8-bit format."""
import ctypes as C
import os
import subprocess

import pytest
import torch

from seed_amd import lib as L
from seed_amd.kv_cache import KVAttention, KVCache
from tests import _kv_ref as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
E_SHAPE, E_DTYPE, E_ALIGN = -1, -2, -3
FAKE = 0x10000                                            # aligned, never dereferenced on these paths


def _handle(**kw):
    h = L.KVCacheStruct(FAKE, FAKE, FAKE, FAKE, 2 * 64, 64, 4, 64, 2, 128, L.KV_MX8)
    for k, v in kw.items():
        setattr(h, k, v)
    return h


def _append(h, **kw):
    a = dict(qkv=FAKE, ldqkv=(4 + 4) * 128, pos=None, base=0, cos=FAKE, sin=FAKE, max_pos=64, q=FAKE, ldq=4 * 128, B=4, T=1, H=4, past=0,
             lens=None)
    a.update(kw)
    return L.load().seedmi_kv_append(None if h is None else C.byref(h), *a.values(), None)


def _read(h, **kw):
    a = dict(k=FAKE, v=FAKE, B=4, n=8, start=0, starts=None)
    a.update(kw)
    return L.load().seedmi_kv_read(C.byref(h), *a.values(), None)


def _attend(h, p=None, **kw):
    a = dict(plen=0, q=FAKE, ldq=4 * 128, out=FAKE, ldo=4 * 128, B=4, T=1, H=4, kv_len=8, lens=None, kv_max=0, scale=0.1, causal=1, ws=None,
             bytes=0)
    a.update(kw)
    return L.load().seedmi_kv_attention(C.byref(h), None if p is None else C.byref(p), *a.values(), None)


@pytest.mark.parametrize("call", [_append, _read, _attend])
@pytest.mark.parametrize("bad,code", [(dict(k=None), E_SHAPE), (dict(slots=0), E_SHAPE), (dict(rows=0), E_SHAPE), (dict(kv_heads=0), E_SHAPE),
                                      (dict(rows=(1 << 22) + 1), E_SHAPE),
                                      (dict(head_dim=96), E_SHAPE), (dict(format=2), E_DTYPE), (dict(k_scale=None), E_SHAPE),
                                      (dict(format=L.KV_16BIT), E_SHAPE), (dict(v=FAKE + 8), E_ALIGN), (dict(v_scale=FAKE + 2), E_ALIGN),
                                      (dict(v_scale=FAKE + 1, head_dim=64), E_ALIGN),
                                      (dict(head_rows=-1), E_SHAPE), (dict(slot_rows=-64), E_SHAPE)])
def test_bad_handles_are_refused(call, bad, code):
    assert call(_handle(**bad)) == code
    assert L.load().seedmi_last_error()


@pytest.mark.parametrize("kw,code", [(dict(B=5), E_SHAPE), (dict(B=0), E_SHAPE), (dict(T=0), E_SHAPE), (dict(past=64), E_SHAPE),
                                     (dict(past=-1), E_SHAPE), (dict(T=65), E_SHAPE), (dict(ldqkv=1016), E_SHAPE), (dict(ldq=504), E_SHAPE),
                                     (dict(ldqkv=1028), E_ALIGN), (dict(ldq=516), E_ALIGN), (dict(max_pos=0), E_SHAPE), (dict(cos=None), E_SHAPE),
                                     (dict(q=FAKE + 4), E_ALIGN), (dict(lens=FAKE + 2), E_ALIGN), (dict(base=-1), E_SHAPE),
                                     (dict(T=1 << 24, lens=FAKE), E_SHAPE)])
def test_append_refuses(kw, code):
    assert _append(_handle(), **kw) == code


def test_append_refuses_overlapping_rows_and_null():
    assert _append(None) == E_SHAPE
    assert _append(_handle(slot_rows=0)) == E_SHAPE
    assert _append(_handle(head_rows=63)) == E_SHAPE
    assert "overlap" in L.load().seedmi_last_error().decode()


@pytest.mark.parametrize("kw,code", [(dict(B=5), E_SHAPE), (dict(n=-1), E_SHAPE), (dict(start=60), E_SHAPE), (dict(start=-1), E_SHAPE),
                                     (dict(k=None, v=None), E_SHAPE), (dict(k=FAKE + 8), E_ALIGN)])
def test_read_refuses(kw, code):
    assert _read(_handle(), **kw) == code


def test_read_of_no_rows_is_nothing_and_16_bit_rows_are_refused():
    assert _read(_handle(), n=0) == 0 and _read(_handle(), n=0, k=None, v=None) == 0
    assert _read(_handle(format=L.KV_16BIT, k_scale=None, v_scale=None)) == E_DTYPE


@pytest.mark.parametrize("kw,code", [(dict(B=5), E_SHAPE), (dict(T=0), E_SHAPE), (dict(H=3), E_SHAPE), (dict(kv_len=65), E_SHAPE),
                                     (dict(kv_len=-1), E_SHAPE), (dict(ldq=504), E_SHAPE), (dict(ldo=504), E_SHAPE), (dict(ldo=516), E_ALIGN),
                                     (dict(q=FAKE + 8), E_ALIGN), (dict(kv_max=-1), E_SHAPE), (dict(scale=float("nan")), E_SHAPE),
                                     (dict(plen=1), E_SHAPE), (dict(plen=-1), E_SHAPE), (dict(T=1 << 28), E_SHAPE),
                                     (dict(kv_len=65, lens=FAKE), E_SHAPE)])
def test_attention_refuses(kw, code):
    assert _attend(_handle(), **kw) == code


def test_attention_refuses_a_prefix_that_does_not_fit():
    ok = dict(slots=1)
    for bad in (dict(head_dim=64), dict(kv_heads=1), dict(format=L.KV_16BIT, k_scale=None, v_scale=None), dict(rows=31)):
        assert _attend(_handle(), _handle(**ok, **bad), plen=32) == E_SHAPE


def test_attention_refuses_more_threads_than_a_launch_has():
    h = _handle(slots=1 << 24)
    assert _attend(h, B=1 << 24) == E_SHAPE and "2^32" in L.load().seedmi_last_error().decode()


def test_attention_refuses_a_short_workspace():
    h = _handle(rows=1 << 20, slot_rows=2 << 20, head_rows=1 << 20)
    need = L.load().seedmi_kv_attention_workspace_bytes(C.byref(h), 1, 1, 4, 0, 0)
    if need:
        assert _attend(h, B=1, kv_len=1 << 20) == E_ALIGN
        assert _attend(h, B=1, kv_len=1 << 20, ws=FAKE, bytes=need - 1) == E_ALIGN
        assert _attend(h, B=1, kv_len=1 << 20, ws=FAKE + 128, bytes=need) == E_ALIGN
    for args in ((0, 1, 4, 0, 0), (1, 0, 4, 0, 0), (1, 1, 3, 0, 0), (1, 1, 4, -1, 0), (1, 1, 4, 0, -1), (5, 1, 4, 0, 0)):
        assert L.load().seedmi_kv_attention_workspace_bytes(C.byref(h), *args) == 0
    assert L.load().seedmi_kv_attention_workspace_bytes(None, 1, 1, 4, 0, 0) == 0


def test_workspace_init_refuses():
    init = L.load().seedmi_kv_attention_workspace_init
    assert init(None, 0, None) == 0
    assert init(None, 8192, None) == E_ALIGN and init(FAKE, 4095, None) == E_ALIGN and init(FAKE + 128, 8192, None) == E_ALIGN


def test_llama_forward_kv_refuses():
    f = L.load().seedmi_llama_forward_kv
    w = L.LlamaWeights()
    w.hidden, w.layers, w.heads, w.max_pos = 256, 1, 2, 64
    kv = (L.KVCacheStruct * 1)(_handle())
    args = dict(w=C.byref(w), kv=kv, prefix=None, plen=0, ids=FAKE, batch=4, T=2, past=FAKE, past_max=8, last=0, logits=FAKE, ldl=64, aws=None, ab=0,
                ws=FAKE, wb=0)
    for bad in (dict(w=None), dict(kv=None), dict(ids=None), dict(past=None), dict(batch=0), dict(batch=5), dict(T=0), dict(past_max=-1),
                dict(past_max=63), dict(plen=1), dict(plen=-1), dict(plen=60, prefix=kv)):
        assert f(*dict(args, **bad).values(), None) == E_SHAPE, bad
    w.heads = 4
    assert f(*args.values(), None) == E_SHAPE                                      # another number of heads than the caches


def test_layout_of_the_handle(tmp_path):
    """The struct of include/seedmi.h, compiled as plain C, against its ctypes mirror."""
    fields = [f for f, _ in L.KVCacheStruct._fields_]
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "seedmi.h"', "int main(void) {",
             '  printf("%zu\\n", sizeof(seedmi_kv_cache_t));']
    lines += [f'  printf("%zu %zu\\n", offsetof(seedmi_kv_cache_t, {f}), sizeof(((seedmi_kv_cache_t*)0)->{f}));' for f in fields]
    (tmp_path / "l.c").write_text("\n".join(lines + ["  return 0;", "}"]))
    subprocess.check_call(["gcc", "-std=c99", "-Wall", "-Werror", "-pedantic", "-I", os.path.join(ROOT, "include"), str(tmp_path / "l.c"),
                           "-o", str(tmp_path / "l")])
    got = subprocess.run([str(tmp_path / "l")], capture_output=True, text=True, check=True).stdout.split("\n")
    assert int(got[0]) == C.sizeof(L.KVCacheStruct)
    for f, line in zip(fields, got[1:]):
        d = getattr(L.KVCacheStruct, f)
        assert line == f"{d.offset} {d.size}", f
    header = open(os.path.join(ROOT, "include", "seedmi.h")).read()
    assert f"#define SEEDMI_KV_16BIT {L.KV_16BIT} " in header and f"#define SEEDMI_KV_MX8 {L.KV_MX8} " in header


def test_python_classes_refuse():
    z = lambda *s, dt=torch.uint8: torch.zeros(*s, dtype=dt)  # noqa: E731
    code, sc = z(2, 2, 8, 128), z(2, 2, 8, 4)
    with pytest.raises(L.SeedmiError, match="HIP device"):
        KVCache.wrap(code, code, sc, sc, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="for both"):
        KVCache.wrap(code, code, sc, None, dtype=torch.bfloat16)
    with pytest.raises(L.SeedmiError, match="bfloat16 or float16"):
        KVCache.wrap(code, code, sc, sc)
    with pytest.raises(ValueError, match="alike"):
        KVCache.wrap(code, z(2, 2, 9, 128), sc, sc, dtype=torch.bfloat16)
    with pytest.raises(L.SeedmiError, match="head_dim 96"):
        KVCache.wrap(z(2, 2, 8, 96), z(2, 2, 8, 96), z(2, 2, 8, 3), z(2, 2, 8, 3), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="scale bytes must be uint8"):
        KVCache.wrap(code, code, z(2, 2, 8, 2), z(2, 2, 8, 2), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="holds torch.float16"):
        KVCache.wrap(code, code, None, None, dtype=torch.float16)
    with pytest.raises(ValueError, match="contiguous and follow"):
        KVCache.wrap(z(2, 2, 128, 8).transpose(2, 3), z(2, 2, 128, 8).transpose(2, 3), sc, sc, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="laid out like"):
        KVCache.wrap(z(2, 2, 16, 128)[:, :, :8], z(2, 2, 16, 128)[:, :, :8], sc, sc, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="format"):
        KVCache.new(1, 1, 8, format="int3", device="cpu")
    with pytest.raises(ValueError, match="without a prefix"):
        KVAttention(None, 4, prefix_len=3)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_reference_format_agrees_with_itself_and_with_the_cast(dtype):
    """The 64-bit restatement that the GPU tests use: every finite 16-bit value in a block of its own magnitude is off by at most half an
    e4m3 step, the codes agree with torch's cast, and the largest of a block lands in (224, 448]."""
    x = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(dtype).view(-1, 1).repeat(1, 32)
    code, sc = R.mx_encode(x, R.top(dtype))
    y = R.mx_decode(code, sc)
    fin = torch.isfinite(x)
    want = x.double().clamp(-R.top(dtype), R.top(dtype))
    e = torch.exp2(sc.double() - 127).repeat_interleave(32, -1)
    assert torch.isnan(y[~fin]).all() and torch.isfinite(y[fin]).all()
    assert ((y - want).abs()[fin] <= torch.maximum(want.abs() * 2.0 ** -4, e * 2.0 ** -10)[fin]).all()
    scaled = (want / e)[fin]
    assert scaled.abs().max() <= 448
    assert (scaled.abs()[(want[fin].abs() > 448 * 2.0 ** -126)] > 224).all()
    cast = scaled.float().to(torch.float8_e4m3fn).view(torch.uint8)
    assert torch.equal(cast, code[fin])
    assert torch.isfinite(y.to(dtype)[fin]).all()
