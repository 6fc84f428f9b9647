"""The entry points of the 4-bit cache and of windows with first keys kept reject bad arguments before any launch (no GPU: fake
pointers, never dereferenced); the wrappers refuse what they do not take."""

from __future__ import annotations

import ctypes

import pytest
import torch

P, N = ctypes.c_void_p(256), None
BATCH = dict(kv=P, page_stride=2560, head_stride=1280, pages=9, page=16, table=P, ts=8, cols=8, seqlens=P, cu=P, B=2, N=4)


def _chunk(lib, **change):
    a = dict(q=P, qs=512, **BATCH, Hq=8, Hkv=2, hd=64, scale=0.125, causal=1, window=0, sinks=0, max_new=0, gate=N, gs=0, out=P,
             os=512, lse=N, ws=N, wb=0, stream=N)
    a.update(change)
    return lib.zb_gqa_chunk_q4(*a.values())


def _append(lib, **change):
    a = dict(proj=P, ps=768, temp=P, positions=N, eps=1e-6, normalize=1, theta=1e4, rotary=64, interleaved=1, q=P, qs=512, **BATCH,
             Hq=8, Hkv=2, hd=64, stream=N)
    a.update(change)
    return lib.zb_gqa_append_q4(*a.values())


def _read(lib, **change):
    a = dict(**BATCH, Hkv=2, hd=64, k=P, ks=128, v=P, vs=128, stream=N)
    a.update(change)
    return lib.zb_kv_read_q4(*a.values())


def _sinks(lib, **change):
    a = dict(q=P, qs=512, k=P, v=P, page_stride=2048, slot_stride=128, head_stride=64, pages=9, page=16, table=P, ts=8, cols=8,
             seqlens=P, cu=P, B=2, N=4, Hq=8, Hkv=2, hd=64, scale=0.125, causal=1, window=9, sinks=2, gate=N, gs=0, out=P, os=512,
             lse=N, ws=N, wb=0, stream=N)
    a.update(change)
    return lib.zb_gqa_chunk_sinks(*a.values())


SHARED = [dict(B=-1), dict(N=-1), dict(Hkv=0), dict(page=0), dict(page=8), dict(page=24), dict(page=1 << 29), dict(page_stride=2552),
          dict(page_stride=-2560), dict(head_stride=1272), dict(ts=7), dict(cu=N), dict(seqlens=N), dict(table=N), dict(kv=N),
          dict(kv=ctypes.c_void_p(264)), dict(B=0), dict(pages=-1)]


@pytest.mark.parametrize("change", SHARED + [dict(Hq=7), dict(Hq=0), dict(scale=0.0), dict(scale=float("inf")), dict(window=-2),
                                             dict(sinks=-1), dict(max_new=-1), dict(causal=0, window=5), dict(qs=504),
                                             dict(qs=516), dict(os=8), dict(q=N), dict(out=ctypes.c_void_p(258)),
                                             dict(gate=P, gs=4)])
def test_chunk_rejects(zb, change):
    assert _chunk(zb._lib.load(), **change) == 1 and "gqa_chunk_q4" in zb._lib.last_error()


@pytest.mark.parametrize("change", SHARED + [dict(rotary=72), dict(rotary=12), dict(rotary=24, interleaved=0), dict(theta=0.0),
                                             dict(eps=-1.0), dict(ps=760), dict(qs=500), dict(Hq=-1), dict(proj=N), dict(q=N)])
def test_append_rejects(zb, change):
    assert _append(zb._lib.load(), **change) == 1 and "gqa_append_q4" in zb._lib.last_error()


@pytest.mark.parametrize("change", SHARED + [dict(ks=120), dict(vs=132), dict(k=N), dict(v=N), dict(v=ctypes.c_void_p(258))])
def test_read_rejects(zb, change):
    assert _read(zb._lib.load(), **change) == 1 and "kv_read_q4" in zb._lib.last_error()


@pytest.mark.parametrize("change", [dict(sinks=-1), dict(window=-1), dict(causal=0), dict(page_stride=2044), dict(q=N), dict(B=0)])
def test_sinks_reject(zb, change):
    assert _sinks(zb._lib.load(), **change) == 1


@pytest.mark.parametrize("hd", [0, 8, 16, 48, 160, 256])
def test_head_dims_outside_the_kernels(zb, hd):
    lib = zb._lib.load()
    assert _chunk(lib, hd=hd) == 3 and _append(lib, hd=hd, rotary=0) == 3 and _read(lib, hd=hd) == 3


def test_nothing_to_do_is_no_launch(zb):
    lib = zb._lib.load()
    before = zb._lib.launch_count()
    assert _chunk(lib, N=0) == 0 and _append(lib, N=0) == 0 and _read(lib, N=0) == 0 and _sinks(lib, N=0) == 0
    assert _chunk(lib, N=0, B=0) == 0 and zb._lib.launch_count() == before


def test_ops_refuse_cpu_tensors_and_shapes(zb):
    ops = zb.ops
    q = torch.zeros(1, 4, 64, dtype=torch.bfloat16)
    cache = ops.kv_q4_cache(2, 16, 2, 64, "cpu")
    assert cache.shape == (2, 2, 1, 1280) and ops.kv_q4_block_bytes(128) == 2560
    table, seqlens, cu = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32), torch.tensor([0, 1], dtype=torch.int32)
    for call in (lambda: ops.gqa_chunk_q4(q, cache, table, seqlens, cu), lambda: ops.kv_read_q4(cache, table, seqlens, cu, 1),
                 lambda: ops.gqa_append_q4(q.flatten(1), cache, table, seqlens, cu, heads=0, kv_heads=2)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    for page, hd in ((8, 64), (0, 64), (20, 64), (16, 48), (16, 256)):
        with pytest.raises(ValueError):
            ops.kv_q4_cache(2, page, 2, hd, "cpu")
