"""The batch entries (include/dflash_batch.h) refuse bad arguments with the documented statuses
before any CUDA call, and the binding refuses tensors that do not fit.  No GPU needed."""
from __future__ import annotations

import ctypes
from types import SimpleNamespace

import pytest
import torch

FAKE = 0x10000  # never dereferenced by these calls


def desc(dc, k=FAKE, ks=FAKE, kb=FAKE, v=FAKE, vs=FAKE, vb=FAKE, S=2, hkv=4, max_len=64, d=64, bits=8, group=64):
    return dc.KVCacheDesc(k, ks, kb, v, vs, vb, S, hkv, max_len, d, bits, group)


BAD_CACHE = [
    (dict(k=0), 1), (dict(v=0), 1), (dict(S=0), 1), (dict(hkv=0), 1), (dict(max_len=0), 1), (dict(d=96), 2),
    (dict(d=512), 2), (dict(bits=3), 2), (dict(bits=0), 2), (dict(group=16), 2), (dict(group=96), 2),
    (dict(d=64, group=128), 2), (dict(ks=0), 1), (dict(vb=0), 1), (dict(k=FAKE + 8), 3), (dict(vs=FAKE + 2), 3),
    (dict(S=65536), 2),
]


def prep(dc, c, qkv=FAKE, ld=2 * 8 * 64 + 2 * 4 * 64, qn=FAKE, kn=FAKE, q_out=FAKE, ld_q=8 * 64, lengths=FAKE, T=4,
         hq=8, rot=64, pos0=0, theta=1e4, parents=None):
    return dc.lib.dflash_stack_attn_prep_batch(qkv, ld, qn, kn, q_out, ld_q, ctypes.byref(c), lengths, T, hq, rot, pos0,
                                               1e-6, theta, parents, None)


def decode(dc, c, q=FAKE, ld_q=8 * 64, gate=FAKE, ld_gate=8 * 64, lengths=FAKE, prefix=None, P=0, out=FAKE, T=4, hq=8,
           parents=None, ws=FAKE, ws_bytes=1 << 40):
    p = None if prefix is None else ctypes.byref(prefix)
    return dc.lib.dflash_stack_attn_decode_batch(q, ld_q, gate, ld_gate, ctypes.byref(c), lengths, p, P, out, T, hq, 0.1,
                                                 parents, ws, ws_bytes, None)


@pytest.mark.parametrize("kw,status", BAD_CACHE)
def test_every_entry_refuses_a_bad_cache(dc, kw, status):
    c = desc(dc, **kw)
    ref = ctypes.byref(c)
    assert prep(dc, c) == status
    assert decode(dc, c) == status
    assert dc.lib.dflash_stack_kv_read(ref, None, 4, FAKE, FAKE, None) == status
    assert dc.lib.dflash_stack_kv_write(ref, None, 4, FAKE, FAKE, None) == status
    assert dc.lib.dflash_stack_kv_compact_batch(ref, FAKE, FAKE, FAKE, 4, None) == status
    assert dc.lib.dflash_stack_attn_decode_batch_workspace_bytes(ref, 0, 4, 8) == 0
    assert dc.last_error()


@pytest.mark.parametrize("kw,status", [
    (dict(qkv=0), 1), (dict(qn=0), 1), (dict(kn=0), 1), (dict(q_out=0), 1), (dict(lengths=0), 1), (dict(T=0), 1),
    (dict(T=65), 1), (dict(hq=0), 1), (dict(pos0=-1), 1), (dict(theta=0.0), 1), (dict(theta=float("nan")), 1),
    (dict(T=33, parents=FAKE), 1), (dict(rot=32), 2), (dict(rot=192), 2), (dict(rot=-64), 2), (dict(ld=1528), 1),
    (dict(ld_q=504), 1), (dict(qkv=FAKE + 2), 3), (dict(ld=1540), 3), (dict(q_out=FAKE + 4), 3), (dict(ld_q=516), 3),
    (dict(qn=FAKE + 2), 3), (dict(pos0=2 ** 31 - 1), 2),
])
def test_prep_argument_errors(dc, kw, status):
    assert prep(dc, desc(dc), **kw) == status


@pytest.mark.parametrize("kw,status", [
    (dict(q=0), 1), (dict(lengths=0), 1), (dict(out=0), 1), (dict(T=0), 1), (dict(T=65), 1), (dict(hq=6), 1),
    (dict(hq=0), 1), (dict(P=-1), 1), (dict(P=5), 1), (dict(T=33, parents=FAKE), 1), (dict(ld_q=504), 1),
    (dict(ld_gate=504), 1), (dict(hq=4 * 65, ld_q=65536, ld_gate=65536), 2), (dict(q=FAKE + 2), 3),
    (dict(ld_q=516), 3), (dict(gate=FAKE + 8), 3), (dict(ld_gate=516), 3), (dict(out=FAKE + 2), 3), (dict(ws=0), 7),
    (dict(ws_bytes=8), 7), (dict(ws=FAKE + 8), 7),
])
def test_decode_argument_errors(dc, kw, status):
    assert decode(dc, desc(dc), **kw) == status


@pytest.mark.parametrize("kw,status", [
    (dict(S=2), 1), (dict(hkv=2), 1), (dict(d=128), 1), (dict(bits=4), 1), (dict(group=32), 1), (dict(max_len=15), 1),
    (dict(k=0), 1), (dict(k=FAKE + 2), 3), (dict(bits=5), 2),
])
def test_decode_refuses_a_prefix_that_does_not_fit(dc, kw, status):
    assert decode(dc, desc(dc), prefix=desc(dc, **{**dict(S=1), **kw}), P=16) == status


def test_the_workspace_does_not_shrink_with_the_batch(dc):
    f = lambda P=0, T=4, hq=8, **kw: dc.lib.dflash_stack_attn_decode_batch_workspace_bytes(  # noqa: E731
        ctypes.byref(desc(dc, **kw)), P, T, hq)
    assert f() > 0
    assert f(S=64) >= f(S=2) and f(P=4096) >= f() and f(T=16) >= f()
    assert f(hq=6) == 0 and f(T=0) == 0 and f(P=-1) == 0


def test_other_argument_errors(dc):
    ref = ctypes.byref(desc(dc))
    read, write, compact = (getattr(dc.lib, "dflash_stack_kv_" + n) for n in ("read", "write", "compact_batch"))
    assert read(ref, None, 0, FAKE, FAKE, None) == 1 and read(ref, None, 65, FAKE, FAKE, None) == 1
    assert read(ref, None, 4, None, None, None) == 1 and read(ref, None, 4, FAKE + 2, None, None) == 3
    assert write(ref, None, 65, FAKE, FAKE, None) == 1 and write(ref, None, 4, None, FAKE, None) == 1
    assert write(ref, None, 4, FAKE, FAKE + 2, None) == 3
    assert compact(ref, FAKE, FAKE, FAKE, 33, None) == 1 and compact(ref, FAKE, FAKE, FAKE, 0, None) == 1
    assert compact(ref, None, FAKE, FAKE, 4, None) == 1 and compact(ref, FAKE, FAKE, None, 4, None) == 1


@pytest.mark.parametrize("kw,status", [
    (dict(x=0), 1), (dict(vocab=0), 1), (dict(rows=-1), 1), (dict(ld=99), 1), (dict(n=-1), 1), (dict(top=-1), 1),
    (dict(tokens=0), 1), (dict(type=2), 2), (dict(top=33), 2), (dict(vocab=7, ld=7, top=8), 2), (dict(x=FAKE + 1), 3),
    (dict(x=FAKE + 2, type=1), 3), (dict(rows=0), 0), (dict(vocab=2**31 - 100, ld=2**31), 2),
])
def test_logprobs_argument_errors(dc, kw, status):
    a = dict(x=FAKE, type=0, ld=100, rows=4, vocab=100, tokens=FAKE, n=1, top=5)
    a.update(kw)
    assert dc.lib.dflash_logprobs(a["x"], a["type"], a["ld"], a["rows"], a["vocab"], a["tokens"], a["n"], a["top"], FAKE,
                                  FAKE, FAKE, FAKE, None) == status


def test_the_binding_refuses_tensors_that_do_not_fit(dc):
    bf = dict(dtype=torch.bfloat16)
    data, sc = torch.zeros(1, 2, 8, 16, dtype=torch.int32), torch.zeros(1, 2, 8, 1, **bf)
    cache = dc.KVCache.of((data, sc, sc), (data, sc, sc), 8, 64)
    assert (cache.sequences, cache.kv_heads, cache.max_len, cache.head_dim) == (1, 2, 8, 64)
    assert cache.nbytes() == 2 * (8 * 2 * 64 + 2 * 2 * 8 * 2)
    for k in ((data.float(), sc, sc), (data, None, sc), (data, sc.float(), sc), (data, sc[:, :, :4], sc),
              (data.transpose(1, 2), sc, sc), (data[0], sc, sc)):
        with pytest.raises(ValueError):
            dc.KVCache.of(k, (data, sc, sc), 8, 64)
    with pytest.raises(dc.DFlashError):
        dc.KVCache(1, 2, 8, 64, 5, device="cpu")
    with pytest.raises(dc.DFlashError):
        dc.KVCache(1, 2, 8, 64, 8, 128, device="cpu")
    # host tensors never reach the library
    with pytest.raises(ValueError, match="CUDA"):
        dc.logprobs(torch.zeros(2, 8))
    with pytest.raises(ValueError, match="CUDA"):
        dc.stack_attn_decode_batch(torch.zeros(1, 128, **bf), cache, torch.zeros(1, dtype=torch.int32), 0.1)


def test_the_binding_refuses_a_stream_of_another_device(dc):
    """Such a call would run on the tensors' device's current stream instead."""
    stream = SimpleNamespace(device=torch.device("cuda", 1))
    with pytest.raises(ValueError, match="stream"):
        dc._elsewhere(torch.device("cuda", 0), stream)


def test_a_stack_over_batch_caches_counts_its_launches():
    """Attention over them is two kernels a layer, over the single-sequence caches one."""
    import verify_stack as vs
    count = lambda bits: vs.VerifyStack.kernels_per_forward(SimpleNamespace(cfg=vs.TINY, kv_bits=bits))  # noqa: E731
    layers = sum(1 for k in vs.TINY.layer_kinds() if k != "gdn")
    assert layers > 0 and count(8) == count(16) == count(None) + layers
