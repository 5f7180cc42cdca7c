"""Cache operators on the CPU: what the entry points refuse before any launch, and the plain forms that the GPU tests
compare with."""
import ctypes
import math
import os

import pytest
import torch

from oracle import cache as oracle


def lib():
    from flint_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    return _lib, _lib.load()


def test_oracle_attention_is_softmax():
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(2, n, h, 64, generator=g, dtype=torch.float64) for n, h in ((3, 4), (2, 9), (2, 9)))
    pos = [6, 2]
    o, lse = oracle.tree_attention(q, k, v, pos, None, 0.125)
    for b in range(2):
        for i in range(3):
            n = pos[b] + i + 1
            for h in range(4):
                s = k[b, h // 2, :n] @ q[b, i, h] * 0.125
                assert torch.allclose(o[b, i, h], torch.softmax(s, 0) @ v[b, h // 2, :n])
                assert torch.allclose(lse[b, i, h], torch.logsumexp(s, 0))
    w = oracle.attention_weights(q, k, lse, pos, None, 0.125)
    assert torch.allclose(w.sum(-1), torch.full((2, 2), 6.0, dtype=torch.float64))
    none = torch.zeros(3, 3, dtype=torch.bool)
    o, lse = oracle.tree_attention(q, k, v, [0, 0], none, 0.125)
    assert (o == 0).all() and (lse == -math.inf).all()


def test_oracle_kept_slots():
    w = [0.5, 0.0, 0.7, 0.0, math.nan, 0.7, 0.1, -1.0]
    assert oracle.kept_slots(w, 8, 3, 0, 0) == [2, 4, 5]
    assert oracle.kept_slots(w, 8, 4, 2, 1) == [0, 4, 6, 7]
    assert oracle.kept_slots(w, 4, 3, 0, 0) == [0, 1, 2]  # equal ones: the lower slot
    assert oracle.kept_slots(w, 5, 9, 0, 0) == [0, 1, 2, 3, 4]


def test_oracle_accept():
    p = [[0.5, 0.25, 0.25], [0.0, 0.0, 1.0], [1.0, 0.0, 0.0]]
    q = [[0.25, 0.5, 0.25], [0.2, 0.3, 0.5]]
    # 0.9 * 0.5 >= 0.25: node 1 rejected, w = (0.25, 0, 0); the next of a chain hangs below it
    assert oracle.accept(p, q, [0, 1, 2], None, [0, 0.9, 0.0], 0.99) == ([0], 0)
    assert oracle.accept(p, q, [0, 1, 2], None, [0, 0.49, 0.999], 0.5) == ([0, 1, 2], 0)
    # a second child of the root: w = (0.25, 0, 0), Z = 0.25
    assert oracle.accept(p, q, [0, 1, 0], [-1, 0, 0], [0, 0.9, 0.99], 0.5) == ([0, 2], 0)
    assert oracle.accept(p, None, [0, 1, 0], [-1, 0, 0], [0, 0.3, 0.7], 0.5) == ([0], 2)


def test_c_entries_refuse():
    _lib, l = lib()
    P = 4096

    def desc(**kw):
        d = _lib.AttnDesc(b=1, m=2, heads=4, groups=2, dim=64, slots=16, fp16=0, pos0=3, scale=0.125, q_b=512, q_m=256, q_h=64,
                          k_b=2048, k_g=1024, k_s=64, v_b=2048, v_g=1024, v_s=64, mask_b=0)
        for k, x in kw.items():
            setattr(d, k, x)
        return ctypes.byref(d)
    need = ctypes.c_int64(-1)
    assert l.fl_tree_attention_workspace(desc(), 1, ctypes.byref(need)) == 0 and need.value >= 0
    bad = [dict(b=0), dict(m=0), dict(heads=3), dict(groups=0), dict(dim=80), dict(slots=1), dict(scale=0.0), dict(scale=-1.0),
           dict(scale=math.nan), dict(scale=math.inf), dict(q_m=4), dict(k_s=1), dict(k_s=1 << 24), dict(v_g=-8), dict(mask_b=-1),
           dict(m=40000, slots=50000)]
    for kw in bad:
        assert l.fl_tree_attention_workspace(desc(**kw), 1, ctypes.byref(need)) == -1, kw
        assert l.fl_tree_attention(desc(**kw), P, P, P, None, None, P, None, P, None) == -1, kw
        assert l.fl_attention_weights(desc(**kw), P, P, P, None, None, P, 0, None) == -1, kw
    for pos in (-1, 15):
        assert l.fl_tree_attention_workspace(desc(pos0=pos), 1, ctypes.byref(need)) == -2
        assert l.fl_tree_attention(desc(pos0=pos), P, P, P, None, None, P, None, P, None) == -2
        assert l.fl_attention_weights(desc(pos0=pos), P, P, P, None, None, P, 0, None) == -2
    for args in ((None, P, P, P), (P, None, P, P), (P, P, None, P), (P, P, P, None), (P + 8, P, P, P), (P, P + 2, P, P)):
        assert l.fl_tree_attention(desc(), *args[:3], None, None, args[3], None, P, None) == -1
    assert l.fl_attention_weights(desc(), P, P, None, None, None, P, 0, None) == -1
    assert l.fl_attention_weights(desc(), P, P, P, None, None, None, 0, None) == -1

    def rows(data=P, outer=2048, inner=1024, row=128):
        return ctypes.byref(_lib.Rows(data, outer, inner, row))

    def evict(k=rows(), v=rows(data=2 * P), w=P, n0=1, n1=2, slots=16, rb=128, n=10, keep=5, recent=1, sink=1, kept=P, ko=None, vo=None, wo=None, so=0):
        return l.fl_evict(k, v, w, n0, n1, slots, rb, n, keep, recent, sink, kept, ko, vo, wo, so, None)
    ko, vo = rows(data=3 * P), rows(data=4 * P)
    for kw in (dict(w=None), dict(kept=None), dict(n0=0), dict(n0=70000), dict(rb=24), dict(rb=8192), dict(n=17), dict(keep=0), dict(keep=11),
               dict(recent=5), dict(recent=-1), dict(sink=-1), dict(k=rows(data=0)), dict(k=rows(data=P + 8)), dict(v=rows(data=2 * P, row=64)),
               dict(v=rows(data=2 * P, inner=8)), dict(v=rows()), dict(k=rows(inner=0)), dict(ko=ko), dict(wo=P), dict(ko=ko, vo=vo, so=4),
               dict(ko=ko, vo=rows(data=4 * P, row=8), so=8), dict(ko=ko, vo=ko, so=8), dict(ko=ko, vo=rows(data=4 * P, inner=0), so=8)):
        assert evict(**kw) == -1, kw

    def accept(p=P, t=P, ua=P, us=P, path=P, b=1, m=2, v=10):
        return l.fl_accept(p, None, 0, t, None, ua, us, path, P, P, b, m, v, None)
    for kw in (dict(p=None), dict(t=None), dict(ua=None), dict(us=None), dict(path=None), dict(b=0), dict(b=70000), dict(m=0), dict(m=1025),
               dict(v=0), dict(v=(1 << 20) + 1)):
        assert accept(**kw) == -1, kw


def test_python_entries_refuse():
    """Everything that is not on a GPU, and shapes and types that do not fit (meta tensors stand for the device)."""
    from flint_amd.attention import attention_weights, evict, tree_attention
    from flint_amd.spec import accept_sampled
    bf = dict(dtype=torch.bfloat16)
    q, k = torch.zeros(1, 2, 4, 64, **bf), torch.zeros(1, 2, 16, 64, **bf)
    with pytest.raises(ValueError, match="CUDA"):
        tree_attention(q, k, k, 3)
    with pytest.raises(ValueError, match="CUDA"):
        attention_weights(q, k, torch.zeros(1, 2, 4), 3)
    with pytest.raises(ValueError):
        evict(k, k, torch.zeros(1, 2, 16), 10, 5)
    with pytest.raises(ValueError, match="one shape"):
        evict(k, k[..., :8, :], torch.zeros(1, 2, 16), 10, 5)
    with pytest.raises(ValueError, match="CUDA"):
        accept_sampled(torch.zeros(1, 2, 9), torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, 2), torch.zeros(1))


def test_more_than_a_launch_holds():
    """2^32 threads and more are refused before a launch."""
    _lib, l = lib()
    P = 4096
    d = _lib.AttnDesc(b=65536, m=1, heads=256, groups=256, dim=64, slots=1, fp16=0, pos0=0, scale=0.125, q_h=64, k_g=64, v_g=64)
    assert l.fl_tree_attention(ctypes.byref(d), P, P, P, None, None, P, None, P, None) == -1
    assert l.fl_attention_weights(ctypes.byref(d), P, P, P, None, None, P, 0, None) == -1
    d = _lib.AttnDesc(b=16, m=40, heads=16, groups=16, dim=64, slots=1 << 30, fp16=0, pos0=0, scale=0.125, q_m=1024, q_h=64, k_s=64, v_s=64)
    assert l.fl_attention_weights(ctypes.byref(d), P, P, P, None, None, P, 0, None) == -1
    r = [ctypes.byref(_lib.Rows(i * P, 0, 0, 4096)) for i in range(1, 5)]
    n = 1 << 25
    assert l.fl_evict(r[0], r[1], P, 1, 1, n, 4096, n, n, 0, 0, P, r[2], r[3], None, n, None) == -1
