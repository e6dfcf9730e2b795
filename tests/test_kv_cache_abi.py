"""include/kf_cache.h and kf_qk_norm_rope without a GPU: symbols, argument checks, and the oracle's own format."""
from __future__ import annotations

import ctypes
import os
import re

import numpy as np

from conftest import REPO
from oracle import q4_oracle as qo

FAKE, MISALIGNED = ctypes.c_void_p(0x10000), ctypes.c_void_p(0x10008)


def test_cache_header_symbols(kf_lib):
    from kernelfoundry_b200 import _lib

    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(REPO, "include", "kf_cache.h")).read(), flags=re.S)
    declared = sorted(set(re.findall(r"\b(kf_[a-z_0-9]+)\s*\(", text)))
    assert declared == sorted(_lib.EXPORTED_CACHE)
    for s in declared:
        assert hasattr(kf_lib, s)


def _strides(*st):
    return (ctypes.c_longlong * len(st))(*st)


def _io(fn, a=FAKE, b=FAKE, c=FAKE, d=FAKE, B=1, S=4, H=2, D=128, nb=4, bs=16, st=(1024, 512, 128), vst=None, flags=0):
    return fn(a, b, c, d, B, S, H, D, nb, bs, _strides(*st, *(vst or st)), flags, None)


def test_write_and_read_arguments(kf_lib):
    from kernelfoundry_b200 import _lib as L

    for fn in (kf_lib.kf_kv_write_q4, kf_lib.kf_kv_read_q4):
        assert _io(fn, D=96) == _io(fn, D=16) == L.KF_ERR_UNSUPPORTED_HEAD_DIM
        for kw in (dict(bs=24), dict(bs=8), dict(bs=512), dict(nb=0), dict(H=0), dict(B=-1), dict(S=-1), dict(flags=2),
                   dict(st=(1024, 512, 100)), dict(vst=(-1024, 512, 128), B=2), dict(a=None), dict(d=None)):
            assert _io(fn, **kw) == L.KF_ERR_INVALID_ARG, kw
        assert _io(fn, B=0) == _io(fn, S=0) == L.KF_OK
    assert _io(kf_lib.kf_kv_write_q4, a=MISALIGNED) == _io(kf_lib.kf_kv_write_q4, c=MISALIGNED) == L.KF_ERR_MISALIGNED
    assert _io(kf_lib.kf_kv_read_q4, a=MISALIGNED) == _io(kf_lib.kf_kv_read_q4, c=MISALIGNED) == L.KF_ERR_MISALIGNED


def test_attention_arguments(kf_lib):
    from kernelfoundry_b200 import _lib as L

    def call(q=FAKE, c=FAKE, o=FAKE, t=FAKE, B=1, Hq=8, Hkv=2, Sq=1, D=128, nb=4, bs=16, mb=4, scale=0.0, flags=0):
        return kf_lib.kf_attn_fwd_paged_q4(q, c, t, FAKE, o, None, None, B, Hq, Hkv, Sq, D, nb, bs, mb, scale, flags, None, 0, None)

    assert call(D=16) == call(D=80) == L.KF_ERR_UNSUPPORTED_HEAD_DIM
    for kw in (dict(Hq=7), dict(Hkv=0), dict(B=-1), dict(Sq=17), dict(bs=48), dict(nb=0), dict(mb=0), dict(flags=16),
               dict(flags=L.KF_FLAG_OUT_F16 | L.KF_FLAG_OUT_BF16), dict(scale=float("inf")), dict(q=None), dict(t=None),
               dict(mb=1 << 27, bs=16)):
        assert call(**kw) == L.KF_ERR_INVALID_ARG, kw
    assert call(q=MISALIGNED) == call(c=MISALIGNED) == call(o=MISALIGNED) == L.KF_ERR_MISALIGNED
    assert call(B=0) == call(Sq=0) == L.KF_OK


def test_qk_norm_rope_arguments(kf_lib):
    from kernelfoundry_b200 import _lib as L

    def call(q=FAKE, k=FAKE, qw=None, qo_=FAKE, ko_=FAKE, B=2, S=4, Hq=4, Hkv=2, D=128, rot=128, theta=1e4, sc=1.0, eps=1e-6,
             st=(2048, 512, 128), flags=0):
        return kf_lib.kf_qk_norm_rope(q, k, qw, None, qo_, ko_, None, None, B, S, Hq, Hkv, D, rot, theta, sc, eps,
                                      _strides(*st, *st, *st, *st), flags, None)

    for kw in (dict(D=24), dict(D=528), dict(rot=8), dict(rot=144), dict(rot=-16), dict(theta=0.0), dict(eps=-1.0),
               dict(sc=float("nan")), dict(flags=4), dict(q=None), dict(ko_=None), dict(Hq=0, Hkv=0), dict(B=-1),
               dict(st=(2048, 512, 4)), dict(rot=4, flags=L.KF_ROPE_GPTJ)):
        assert call(**kw) == L.KF_ERR_INVALID_ARG, kw
    assert call(q=MISALIGNED) == call(ko_=MISALIGNED) == call(qw=MISALIGNED) == L.KF_ERR_MISALIGNED
    assert call(B=0) == call(S=0) == L.KF_OK


def test_oracle_quantiser_holds_its_bound():
    """Half a step, zero exact, the row's sign structure, and pack/unpack as the header says."""
    rng = np.random.default_rng(1)
    x = (rng.standard_normal((50, 64)) * 10.0 ** rng.uniform(-6, 4, (50, 1)) + rng.choice([0, 5.0], (50, 1))).astype(np.float32)
    n, w = qo.quantise(x)
    step = (np.maximum(x.max(-1), 0) - np.minimum(x.min(-1), 0)) / 15
    assert (np.abs(qo.values(n, w) - x).max(-1) <= step * (0.5 + 2.0 ** -10)).all()
    assert (qo.values(*qo.quantise(np.zeros((3, 64)))) == 0).all()
    c = qo.write(qo.empty_cache(2, 1, 32, 64), np.array([[37]], np.int32), x[:1].reshape(1, 1, 1, 64), x[1:2].reshape(1, 1, 1, 64))
    g = c[1, 0, 0]                                       # slot 37: block 1, group 0, row 5
    assert g[5 * 32] == n[0, 0] | n[0, 1] << 4 and g[512 + 5 * 32 + 31] == n[1, 62] | n[1, 63] << 4
    assert g[1024:].view(np.uint32)[5] == w[0] and g[1024:].view(np.uint32)[16 + 5] == w[1]
    assert c[0].max() == 0 and c[1, 0, 1].max() == 0


def test_oracle_attention_equals_a_direct_softmax():
    rng = np.random.default_rng(2)
    cache = qo.empty_cache(3, 1, 16, 64)
    k, v = rng.standard_normal((2, 1, 1, 20, 64))
    table = np.array([[2, 0]], np.int32)
    slots = (table[0, np.arange(20) // 16] * 16 + np.arange(20) % 16)[None].astype(np.int32)
    cache = qo.write(cache, slots, k, v)
    kq, vq = (qo.values(*qo.quantise(x[0, 0])) for x in (k, v))
    q = rng.standard_normal((1, 2, 3, 64))
    O, Mi, Li, _ = qo.attention(q, cache, table, [20], causal=True)
    for h, i in np.ndindex(2, 3):
        s = kq[:18 + i] @ q[0, h, i] / 8
        p = np.exp(s - s.max())
        np.testing.assert_allclose(O[0, h, i], p @ vq[:18 + i] / p.sum(), rtol=1e-12)
        assert np.isclose(Mi[0, h, i], s.max()) and np.isclose(Li[0, h, i], p.sum())


def test_workspace_form(kf_lib):
    """A workspace elsewhere, of another type or with gaps never reaches the kernel."""
    import pytest
    import torch

    from kernelfoundry_b200.kv_cache import _check_workspace

    here, there = torch.device("cpu"), torch.device("meta")
    _check_workspace(torch.zeros(64, dtype=torch.uint8), here)
    for ws, dev in ((torch.zeros(64, dtype=torch.uint8), there), (torch.zeros(64, dtype=torch.float32), here),
                    (torch.zeros(128, dtype=torch.uint8)[::2], here)):
        with pytest.raises(ValueError, match="workspace"):
            _check_workspace(ws, dev)
