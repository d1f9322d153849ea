"""What the rotary, append and shared-prefix operators refuse, on the host: wrong arguments never reach a launch. Frequency tables."""
import ctypes
import math

import pytest
import torch

from volundr_mlx_b200 import _lib, build, ops, rotary


@pytest.fixture(scope="module")
def L():
    build.build()
    return _lib.lib()


def test_frequencies():
    f, m = rotary.frequencies(8, 1e4)
    assert f.dtype == torch.float64 and m == 1.0 and torch.allclose(f, torch.tensor([1, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-15)
    assert torch.equal(rotary.frequencies(8, 1e4, scaling="linear", factor=4.0)[0], f / 4)
    n = rotary.frequencies(8, 1e4, scaling="ntk", factor=4.0)[0]
    assert n[0] == 1.0 and abs(float(n[-1] / f[-1]) - 0.25) < 1e-14        # fastest kept, slowest divided
    p, m = rotary.frequencies(64, 1e4, scaling="parts", factor=8.0, trained_len=4096)
    f = rotary.frequencies(64, 1e4)[0]
    turns = 4096 * f / (2 * math.pi)
    assert torch.equal(p[turns > 32], f[turns > 32]) and torch.allclose(p[turns < 1], f[turns < 1] / 8, rtol=1e-15)
    assert bool((p <= f).all()) and bool((p >= f / 8 * (1 - 1e-15)).all()) and abs(m - (0.1 * math.log(8) + 1)) < 1e-15
    assert rotary.frequencies(64, 1e4, scaling="parts", factor=8.0, magnitude=1.0)[1] == 1.0
    assert rotary.frequencies(0, 1e4)[0].numel() == 0
    for bad in (dict(dims=3), dict(dims=-2), dict(theta=0.0), dict(factor=0.5), dict(scaling="yes"), dict(scaling="parts", high=1.0)):
        with pytest.raises(ValueError):
            rotary.frequencies(**{"dims": 8, "theta": 1e4, **bad})


def test_wrappers_refuse_cpu_tensors():
    x, pos, freq = torch.zeros(2, 3, 64, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32), torch.ones(32, dtype=torch.float64)
    pages = torch.zeros(4, 3, 64, 64, dtype=torch.bfloat16)
    table, one = torch.zeros(2, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.rope(x, pos, freq)
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv_append(x, x, pages, pages, table, pos, freq)
    with pytest.raises(ValueError, match="CUDA"):
        ops.attend_prefix(x, pages, pages, one, one, table, pos)


A = 0x10000   # an address that no refused call may touch


def rope_args(**kw):
    a = _lib.RopeArgs()
    d = dict(dtype=0, rows=4, heads=2, D=64, dims=64, interleaved=0, inverse=0, magnitude=1.0, x=A, x_row=128, x_head=64, out=A, out_row=128,
             out_head=64, pos=A, freq=A)
    d.update(kw)
    for k, v in d.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad", [dict(dtype=2), dict(dtype=-1), dict(dims=3), dict(dims=66), dict(dims=-2), dict(D=0), dict(D=1026, dims=2),
                                 dict(rows=-1), dict(heads=0), dict(x=None), dict(out=None), dict(pos=None), dict(freq=None), dict(x=A + 1),
                                 dict(out_row=10), dict(out_head=10), dict(x_row=-1), dict(x_head=-1), dict(magnitude=math.nan)])
def test_rope_refuses(L, bad):
    assert L.vk_rope(ctypes.byref(rope_args(**bad)), None) == -1
    assert L.vk_rope(ctypes.byref(rope_args(rows=0)), None) == 0
    assert L.vk_rope(None, None) == -1


def append_args(**kw):
    a = _lib.AppendArgs()
    d = dict(dtype=0, rows=4, Hq=2, KVH=2, D=64, dims=64, interleaved=0, magnitude=1.0, q=A, k=A, v=A, q_row=128, q_head=64, k_row=128,
             k_head=64, v_row=128, v_head=64, q_out=A, qo_row=128, qo_head=64, K=A, V=A, table=A, pos=A, slot=None, seq=None, freq=A,
             n_seqs=4, max_pages=2, n_pages=9)
    d.update(kw)
    for k, v in d.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad", [dict(dtype=3), dict(dims=5), dict(dims=128), dict(rows=-1), dict(KVH=0), dict(Hq=-1), dict(Hq=0), dict(n_seqs=0),
                                 dict(max_pages=0), dict(n_pages=0), dict(q_out=None), dict(q=None), dict(k=None), dict(v=None),
                                 dict(K=None), dict(V=None), dict(table=None), dict(pos=None), dict(freq=None), dict(rows=5), dict(k=A + 1),
                                 dict(qo_row=1), dict(qo_head=1), dict(v_head=-64)])
def test_append_refuses(L, bad):
    assert L.vk_kv_append(ctypes.byref(append_args(**bad)), None) == -1
    assert L.vk_kv_append(ctypes.byref(append_args(rows=0)), None) == 0
    assert L.vk_kv_append(None, None) == -1


def prefix_args(**kw):
    a = _lib.PrefixArgs()
    d = dict(dtype=0, seqs=4, T=2, Hq=4, KVH=2, D=64, scale=0.1, q=A, q_row=256, q_head=64, gate=None, out=A, out_row=256, out_head=64,
             K=A, V=A, n_pages=9, prefix_pages=A, max_prefix_pages=3, prefix_len=A, table=A, max_pages=2, lens=A)
    d.update(kw)
    for k, v in d.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad", [dict(dtype=2), dict(D=96), dict(D=256), dict(seqs=-1), dict(T=0), dict(Hq=3), dict(KVH=0), dict(scale=0.0),
                                 dict(scale=math.nan), dict(scale=math.inf), dict(scale=-1.0), dict(n_pages=0), dict(max_prefix_pages=-1), dict(max_pages=-1),
                                 dict(prefix_len=None), dict(lens=None), dict(K=None), dict(V=None), dict(q=None), dict(out=None),
                                 dict(prefix_pages=None), dict(table=None), dict(q=A + 2), dict(out=A + 8), dict(K=A + 4), dict(V=A + 4),
                                 dict(gate=A + 2), dict(q_row=252), dict(q_head=60), dict(out_row=8), dict(out_head=63), dict(gate=A, gate_row=3)])
def test_attend_refuses(L, bad):
    a = prefix_args(**bad)
    assert L.vk_attend_prefix(ctypes.byref(a), A, 1 << 40, None) == -1
    assert L.vk_attend_prefix_workspace_bytes(ctypes.byref(a)) == 0


def test_attend_refuses_what_its_indices_cannot_hold(L):
    for bad in (dict(n_pages=1 << 25), dict(max_prefix_pages=1 << 25), dict(max_pages=1 << 25), dict(seqs=65536)):
        assert L.vk_attend_prefix(ctypes.byref(prefix_args(**bad)), A, 1 << 40, None) == -3
    ok = prefix_args()
    need = L.vk_attend_prefix_workspace_bytes(ctypes.byref(ok))
    assert need > 0
    assert L.vk_attend_prefix(ctypes.byref(ok), A, need - 1, None) == -2
    assert L.vk_attend_prefix(ctypes.byref(ok), None, need, None) == -1
    assert L.vk_attend_prefix(ctypes.byref(ok), A + 8, need, None) == -1
    assert L.vk_attend_prefix(ctypes.byref(prefix_args(seqs=0)), A, 16, None) == 0
