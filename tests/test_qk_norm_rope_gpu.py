"""qk_norm_rope (include/kf_pointwise.h) vs the fp64 oracle.

Tolerance: the kernel carries fp32 intermediates (a sum of D squares, rsqrtf, the
products, cos/sin of an angle reduced in fp64) and rounds once.  Each relative error is
a few 2^-24, together below 2^-19, of the pair's magnitude |y0| + |y1| (times the
rotation's scale); the output rounding adds half an ulp, and a rounding boundary
crossed by the fp32 error another half: 1 ulp + 2^-19 (|y0| + |y1|).
"""
from __future__ import annotations

import numpy as np
import pytest

from oracle import pointwise_oracle as po
from oracle import q4_oracle as qo

pytestmark = pytest.mark.gpu


def _dev(a, dt, device):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(device).to(torch.float16 if dt == "f16" else torch.bfloat16)


def _host(t):
    return t.float().cpu().numpy().astype(np.float64)


def _pair_mag(y, rot, interleaved):
    """|y0| + |y1| of each element's pair; |y| where nothing rotates."""
    m = np.abs(y).copy()
    a = np.abs(y[..., :rot])
    if rot and interleaved:
        s = a[..., 0::2] + a[..., 1::2]
        m[..., :rot] = np.repeat(s, 2, -1)
    elif rot:
        s = a[..., :rot // 2] + a[..., rot // 2:]
        m[..., :rot] = np.concatenate((s, s), -1)
    return m


def _check(got, x, w, pos, dt, what, eps=1e-6, theta=10000.0, rot=None, interleaved=False, inv_freq=None, rot_scale=1.0):
    rot = x.shape[-1] if rot is None else rot
    ref, y = qo.qk_norm_rope(x, w, pos, eps, dt, theta, rot, interleaved, inv_freq, rot_scale)
    tol = po.ulp(ref, dt) + 2.0 ** -19 * _pair_mag(y, rot, interleaved) * max(1.0, abs(rot_scale))
    bad = np.abs(got - ref) > tol
    assert np.isfinite(got).all() and not bad.any(), f"{what}: {bad.sum()} outside, worst {(np.abs(got - ref) / tol).max():.2f}x"


CASES = [
    # B, S, H_q, H_kv, D, rot, interleaved, dtype
    (1, 1, 1, 1, 16, 16, False, "f16"),
    (1, 1, 32, 8, 128, 128, False, "bf16"),
    (64, 1, 32, 8, 128, 128, False, "f16"),
    (2, 33, 5, 3, 64, 32, True, "bf16"),
    (3, 17, 7, 1, 256, 64, True, "f16"),
    (2, 9, 10, 5, 96, 96, False, "bf16"),
    (1, 7, 3, 2, 80, 16, False, "f16"),
    (2, 5, 4, 4, 512, 512, False, "f16"),
    (1, 6, 2, 1, 144, 8, True, "bf16"),
    (1, 700, 8, 2, 128, 0, False, "bf16"),
    (5, 1, 16, 0, 128, 64, False, "f16"),
    (1, 2049, 40, 8, 128, 128, False, "bf16"),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "B{}_S{}_Hq{}_Hkv{}_D{}_r{}_{}_{}".format(*c))
def test_qk_norm_rope_matches_oracle(cuda, case):
    import torch

    from kernelfoundry_b200 import qk_norm_rope

    B, S, Hq, Hkv, D, rot, inter, dt = case
    rng = np.random.default_rng(sum(case[:6]))
    q, k = (po.round_to(3 * rng.standard_normal((B, h, S, D)), dt) for h in (Hq, Hkv))
    wq, wk = (po.round_to(1 + 0.3 * rng.standard_normal(D), dt) for _ in range(2))
    pos = rng.integers(0, 2 ** 17, (B, S)).astype(np.int32)
    kt = _dev(k, dt, cuda) if Hkv else None
    qo_, ko_ = qk_norm_rope(_dev(q, dt, cuda), kt, _dev(wq, dt, cuda), _dev(wk, dt, cuda) if Hkv else None,
                            torch.from_numpy(pos).to(cuda), rot_dim=rot, interleaved=inter, theta=500000.0)
    _check(_host(qo_), q, wq, pos, dt, "q", theta=500000.0, rot=rot, interleaved=inter)
    if Hkv:
        _check(_host(ko_), k, wk, pos, dt, "k", theta=500000.0, rot=rot, interleaved=inter)
    else:
        assert ko_ is None


@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_views_of_a_fused_projection_and_storage_order(cuda, dt):
    """Strided [B, S, H, D] views in, [B, H, S, D] storage out, a frequency table, a rotation scale, default positions."""
    import torch

    from kernelfoundry_b200 import qk_norm_rope

    B, S, Hq, Hkv, D = 2, 37, 6, 2, 128
    rng = np.random.default_rng(5)
    qkv = po.round_to(rng.standard_normal((B, S, (Hq + 2 * Hkv) * D)), dt)
    t = _dev(qkv, dt, cuda)
    q, k = t[..., :Hq * D].view(B, S, Hq, D), t[..., Hq * D:(Hq + Hkv) * D].view(B, S, Hkv, D)
    freq = (10000.0 ** (-np.arange(0, D, 2) / D) / np.where(np.arange(D // 2) > 20, 8.0, 1.0)).astype(np.float32)
    q_out, k_out = (torch.empty(B, h, S, D, dtype=t.dtype, device=cuda) for h in (Hq, Hkv))
    res = qk_norm_rope(q, k, None, None, inv_freq=torch.from_numpy(freq).to(cuda), rot_scale=1.25, eps=1e-5, layout="bshd",
                       out=(q_out.transpose(1, 2), k_out.transpose(1, 2)))
    assert res[0].data_ptr() == q_out.data_ptr()
    pos = np.broadcast_to(np.arange(S), (B, S))
    for got, x in ((q_out, qkv[..., :Hq * D].reshape(B, S, Hq, D)), (k_out, qkv[..., Hq * D:(Hq + Hkv) * D].reshape(B, S, Hkv, D))):
        _check(_host(got), x.transpose(0, 2, 1, 3), None, pos, dt, "view", eps=1e-5, inv_freq=freq, rot_scale=1.25)


def test_in_place_equals_out_of_place(cuda):
    import torch

    from kernelfoundry_b200 import qk_norm_rope

    torch.manual_seed(0)
    for inter in (False, True):
        q = torch.randn(3, 50, 9, 128, device=cuda).half()
        k = torch.randn(3, 50, 3, 128, device=cuda).half()
        w = torch.ones(128, device=cuda).half()
        a, b = qk_norm_rope(q, k, w, w, rot_dim=64, interleaved=inter, layout="bshd")
        qk_norm_rope(q, k, w, w, rot_dim=64, interleaved=inter, layout="bshd", out=(q, k))
        assert torch.equal(a, q) and torch.equal(b, k)


def test_extreme_rows(cuda):
    """Zero rows stay zero, a NaN or an infinity spoils its own row only, large and tiny rows keep their direction."""
    import torch

    from kernelfoundry_b200 import qk_norm_rope

    q = torch.ones(1, 6, 1, 128, device=cuda, dtype=torch.bfloat16)
    q[0, 0] = 0
    q[0, 1, 0, 5] = float("nan")
    q[0, 2, 0, 5] = float("inf")
    q[0, 3] = 2.0 ** 60
    q[0, 4] = 2.0 ** -60
    out, _ = qk_norm_rope(q, None, None, None, rot_dim=0)
    out = out.float().cpu()[0, :, 0]
    assert (out[0] == 0).all() and torch.isnan(out[1]).all() and torch.isnan(out[2, 5])
    assert (out[3] == 1).all() and (out[5] == 1).all()
    assert torch.isfinite(out[4]).all()


def test_empty_calls_and_own_stream(cuda):
    import torch

    from kernelfoundry_b200 import qk_norm_rope

    e = torch.empty(0, 4, 3, 64, device=cuda, dtype=torch.float16)
    assert qk_norm_rope(e, e, None, None)[0].shape == e.shape
    torch.manual_seed(1)
    q = torch.randn(4, 8, 100, 64, device=cuda).half()
    want = qk_norm_rope(q, None, None, None)[0]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = qk_norm_rope(q, None, None, None)[0]
    side.synchronize()
    assert torch.equal(got, want)


def test_refusals(cuda):
    import torch

    from kernelfoundry_b200 import KFError, qk_norm_rope

    q = torch.zeros(2, 4, 8, 128, device=cuda, dtype=torch.float16)
    w = torch.ones(128, device=cuda, dtype=torch.float16)
    bad = [
        (dict(q=q.cpu()), ValueError), (dict(q=q.float()), ValueError), (dict(k=q.bfloat16()), ValueError),
        (dict(k=q[:, :, :5]), ValueError), (dict(q_weight=w[:64]), ValueError), (dict(q_weight=w.float()), ValueError),
        (dict(positions=torch.zeros(2, 8, device=cuda)), ValueError), (dict(inv_freq=torch.zeros(3, device=cuda)), ValueError),
        (dict(layout="sbhd"), ValueError), (dict(q=q.transpose(2, 3)), ValueError), (dict(out=(q[:, :2], None)), ValueError),
        (dict(rot_dim=24), KFError), (dict(rot_dim=256, inv_freq=None), KFError), (dict(eps=float("nan")), KFError),
        (dict(theta=-1.0), KFError), (dict(q=torch.zeros(1, 1, 1, 24, device=cuda, dtype=torch.float16), q_weight=None), KFError),
    ]
    for change, err in bad:
        args = dict(q=q, k=None, q_weight=w, k_weight=None)
        args.update(change)
        with pytest.raises(err):
            qk_norm_rope(args.pop("q"), args.pop("k"), args.pop("q_weight"), args.pop("k_weight"), **args)
    odd = torch.zeros(2 * 4 * 8 * 128 + 4, device=cuda, dtype=torch.float16)[4:].view(2, 4, 8, 128)
    with pytest.raises(KFError, match="aligned"):
        qk_norm_rope(odd, None, None, None)
    narrow = torch.zeros(2, 4, 8, 132, device=cuda, dtype=torch.float16)[..., :128]
    with pytest.raises(KFError, match="invalid"):
        qk_norm_rope(narrow, None, None, None)


LARGE = [
    # groups of 8 tokens (4 at D = 512, 2 for 700 sequences), and blocks that go on to a second and a third group
    (1, 2500, 3, 1, 128, 128, False, "f16"),
    (1, 5003, 3, 2, 128, 64, False, "bf16"),
    (2, 4999, 2, 1, 64, 64, True, "f16"),
    (3, 1701, 1, 1, 256, 256, False, "f16"),
    (1, 2417, 1, 1, 512, 512, False, "bf16"),
    (700, 1, 4, 1, 128, 128, False, "f16"),
    (1, 9999, 1, 1, 80, 16, False, "f16"),
    (1, 2400, 41, 3, 96, 96, True, "bf16"),
]


@pytest.mark.parametrize("case", LARGE, ids=lambda c: "B{}_S{}_Hq{}_Hkv{}_D{}_r{}_{}_{}".format(*c))
def test_groups_of_tokens_and_blocks_with_several(cuda, case):
    test_qk_norm_rope_matches_oracle(cuda, case)


def test_groups_of_tokens_in_place_and_out_of_place_agree(cuda):
    """5000 tokens (blocks take two groups): rows read for one group are not what another has written."""
    import torch

    from kernelfoundry_b200 import qk_norm_rope

    torch.manual_seed(6)
    q, k = (torch.randn(1, 5000, h, 128, device=cuda).half() for h in (5, 2))
    a, b = qk_norm_rope(q, k, None, None, layout="bshd")
    qk_norm_rope(q, k, None, None, layout="bshd", out=(q, k))
    assert torch.equal(a, q) and torch.equal(b, k)
