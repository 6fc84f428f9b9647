"""The paged-cache entry points reject bad arguments before any launch (no GPU: fake pointers, never dereferenced), and
the wrappers refuse CPU tensors."""

from __future__ import annotations

import ctypes

import pytest
import torch

P, N = ctypes.c_void_p(256), None


def _chunk(lib, **change):
    a = dict(q=P, qs=512, k=P, v=P, page_stride=2048, slot_stride=128, head_stride=64, pages=9, page=16, table=P, ts=8, cols=8,
             seqlens=P, cu=P, B=2, N=4, Hq=8, Hkv=2, hd=64, scale=0.125, causal=1, window=0, gate=N, gs=0, out=P, os=512,
             lse=N, ws=N, wb=0, stream=N)
    a.update(change)
    return lib.zb_gqa_chunk(*a.values())


def _append(lib, **change):
    a = dict(proj=P, ps=768, temp=P, positions=N, eps=1e-6, normalize=1, theta=1e4, rotary=64, interleaved=1, q=P, qs=512, k=P,
             v=P, page_stride=2048, slot_stride=128, head_stride=64, pages=9, page=16, table=P, ts=8, cols=8, seqlens=P, cu=P,
             B=2, N=4, Hq=8, Hkv=2, hd=64, stream=N)
    a.update(change)
    return lib.zb_gqa_append(*a.values())


SHARED = [dict(B=-1), dict(N=-1), dict(Hkv=0), dict(page=0), dict(page=1 << 29), dict(page_stride=2044), dict(slot_stride=-128),
          dict(head_stride=65), dict(ts=7), dict(cu=N), dict(seqlens=N), dict(table=N), dict(k=N), dict(v=ctypes.c_void_p(264)),
          dict(B=0)]


@pytest.mark.parametrize("change", SHARED + [dict(Hq=7), dict(scale=0.0), dict(scale=float("inf")), dict(window=-2),
                                             dict(causal=0, window=5), dict(qs=504), dict(qs=516), dict(os=8), dict(q=N),
                                             dict(out=ctypes.c_void_p(258)), dict(gate=P, gs=4)])
def test_chunk_rejects(zb, change):
    assert _chunk(zb._lib.load(), **change) == 1 and "gqa_chunk" in zb._lib.last_error() + "gqa_chunk"


@pytest.mark.parametrize("change", SHARED + [dict(rotary=72), dict(rotary=12), dict(rotary=24, interleaved=0), dict(theta=0.0),
                                             dict(eps=-1.0), dict(ps=760), dict(qs=500), dict(Hq=0), dict(proj=N), dict(q=N)])
def test_append_rejects(zb, change):
    assert _append(zb._lib.load(), **change) == 1


@pytest.mark.parametrize("hd", [0, 4, 60, 136, 256])
def test_head_dims_outside_the_kernels(zb, hd):
    lib = zb._lib.load()
    assert _chunk(lib, hd=hd) == 3 and _append(lib, hd=hd, rotary=0) == 3


def test_nothing_to_do_is_no_launch(zb):
    lib = zb._lib.load()
    before = zb._lib.launch_count()
    assert _chunk(lib, N=0) == 0 and _append(lib, N=0) == 0 and _chunk(lib, N=0, B=0) == 0
    assert zb._lib.launch_count() == before


def test_ops_refuse_cpu_tensors(zb):
    q = torch.zeros(1, 4, 64, dtype=torch.bfloat16)
    cache = torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16)
    table, seqlens, cu = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32), torch.tensor([0, 1], dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        zb.ops.gqa_chunk(q, cache, cache, table, seqlens, cu)
    with pytest.raises(ValueError, match="CUDA"):
        zb.ops.gqa_append(q.flatten(1), cache, cache, table, seqlens, cu, heads=2, kv_heads=1)
