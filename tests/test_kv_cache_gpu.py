"""The 4-bit KV cache (include/kf_cache.h): written bytes, values read back, attention, refusals.

Write and read are exact: the quantiser is a fixed sequence of fp32 operations, so the
cache's bytes equal the oracle's, and a read is one rounding of an exact product.

Attention against the oracle in 64 bits (on the values the codes stand for), per element:
the probabilities are rounded to fp16 (relative 2^-11 at most); scores carry fp32 errors
(dot products of 15 * D terms, the scale products: below 2^-18 of |x| with |x| < 40 in
these inputs, so 2^-12.6 at the very most and far less where p matters), the exponential
and the sums below 2^-18: together 2^-10 of A = sum p |v| / l, plus the output's rounding
(half an ulp: 2^-11 or 2^-8 of |O|; 2^-24 for fp32).  Mi: 2^-18 * max(|Mi|, 1); Li: 2^-12.
"""
from __future__ import annotations

import numpy as np
import pytest

from oracle import pointwise_oracle as po
from oracle import q4_oracle as qo

pytestmark = pytest.mark.gpu


def _tdt(dt):
    import torch

    return {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}[dt]


def _dev(a, dt, device):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(device).to(_tdt(dt))


def _host(t):
    return t.float().cpu().numpy().astype(np.float64)


# ------------------------------------------------------------------ write and read
IO = [
    # B, S, H, D, block_size, dtype
    (1, 1, 1, 64, 16, "f16"),
    (16, 1, 8, 128, 16, "f16"),
    (3, 21, 5, 64, 32, "bf16"),
    (2, 100, 3, 256, 64, "f16"),
    (1, 257, 2, 128, 256, "bf16"),
    (2, 333, 8, 128, 128, "f16"),
    (1, 40, 7, 256, 16, "bf16"),
]


@pytest.mark.parametrize("case", IO, ids=lambda c: "B{}_S{}_H{}_D{}_bs{}_{}".format(*c))
@pytest.mark.parametrize("layout", ["bhsd", "bshd"])
def test_write_bytes_and_read_values(cuda, case, layout):
    import torch

    from kernelfoundry_b200 import kv_read_q4, kv_write_q4

    B, S, H, D, bs, dt = case
    rng = np.random.default_rng(sum(case[:5]))
    k, v = (po.round_to(rng.standard_normal((B, H, S, D)) * rng.choice([0.01, 1.0, 30.0], (B, H, S, 1)), dt) for _ in range(2))
    k[0, 0, 0] = 0.0                                     # an all-zero row
    v[-1, -1, -1] = 3.0                                  # a constant row
    v[0, 0, -1] = -np.abs(v[0, 0, -1])                   # a row without positive values
    n_blocks = -(-B * S // bs) + 2
    slots = rng.permutation(n_blocks * bs)[:B * S].reshape(B, S).astype(np.int32)
    if B * S > 3:
        slots[0, 0], slots[-1, -1] = -1, n_blocks * bs   # skipped on write, zeros on read
    start = rng.integers(0, 256, (n_blocks, H, bs // 16, 16 * (D + 8)), dtype=np.uint8)
    cache = torch.from_numpy(start.copy()).to(cuda)
    kt, vt = _dev(k, dt, cuda), _dev(v, dt, cuda)
    if layout == "bshd":
        kt, vt = (x.transpose(1, 2).contiguous() for x in (kt, vt))
    st = torch.from_numpy(slots).to(cuda)
    kv_write_q4(kt, vt, cache, st, layout=layout)
    want = qo.write(start, slots, k, v)
    np.testing.assert_array_equal(cache.cpu().numpy(), want)
    for out_dt in ("f16", "bf16"):
        got = kv_read_q4(cache, st, dtype=_tdt(out_dt), layout=layout)
        for g, r in zip(got, qo.read(want, slots)):
            g = _host(g if layout == "bhsd" else g.transpose(1, 2))
            np.testing.assert_array_equal(g, po.round_to(r, out_dt))
    # what is held is within half a step of what was written
    ok = (slots >= 0) & (slots < n_blocks * bs)
    for x, r in zip((k, v), qo.read(want, slots)):
        step = (np.maximum(x.max(-1), 0) - np.minimum(x.min(-1), 0)) / 15
        err = np.abs(x - r).max(-1) <= step * (0.5 + 2.0 ** -10)
        assert err[np.broadcast_to(ok[:, None], err.shape)].all()


def test_write_strided_views_and_out(cuda):
    """Views of a fused projection in, views of a larger buffer out; K and V strides differ."""
    import torch

    from kernelfoundry_b200 import kv_read_q4, kv_write_q4, q4_cache

    B, S, H, D = 2, 19, 3, 128
    torch.manual_seed(3)
    qkv = torch.randn(B, S, 5 * H * D, device=cuda).half()
    k = qkv[..., 3 * H * D:4 * H * D].view(B, S, H, D)
    v = torch.randn(B, H, S, D, device=cuda).half().transpose(1, 2)
    slots = torch.arange(B * S, device=cuda, dtype=torch.int32).view(B, S)
    cache, plain = q4_cache(3, H, 16, D, cuda), q4_cache(3, H, 16, D, cuda)
    kv_write_q4(k, v, cache, slots, layout="bshd")
    kv_write_q4(k.transpose(1, 2).contiguous(), v.transpose(1, 2).contiguous(), plain, slots)
    assert torch.equal(cache, plain)
    big = torch.full((2, B, S, H, 2 * D), 7.0, device=cuda, dtype=torch.float16)
    outs = (big[0, ..., :D], big[1, ..., D:])
    kv_read_q4(cache, slots, layout="bshd", out=outs)
    want = kv_read_q4(cache, slots, layout="bshd")
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
    assert (big[0, ..., D:] == 7).all() and (big[1, ..., :D] == 7).all()


@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_extreme_rows(cuda, dt):
    """NaN and infinities spoil their own row; the type's largest, smallest and subnormal values keep the bound."""
    import torch

    from kernelfoundry_b200 import kv_read_q4, kv_write_q4

    D, rows = 64, 12
    rng = np.random.default_rng(0)
    top = 65504.0 if dt == "f16" else 3.3895313892515355e38
    tiny = 2.0 ** -24 if dt == "f16" else 2.0 ** -133
    x = po.round_to(rng.standard_normal((1, 1, rows, D)), dt)
    x[0, 0, 0, 3] = np.nan
    x[0, 0, 1, 63] = np.inf
    x[0, 0, 2, 0] = -np.inf
    x[0, 0, 3, :2] = top, -top
    x[0, 0, 4] = tiny
    x[0, 0, 5] = 0.0
    x[0, 0, 6] = -0.0
    x[0, 0, 7] = rng.choice([0.0, tiny], D)
    x[0, 0, 8] = np.nan
    start = np.zeros((1, 1, 1, 16 * (D + 8)), np.uint8)
    slots = np.arange(rows, dtype=np.int32)[None]
    cache = torch.from_numpy(start.copy()).to(cuda)
    xt = torch.from_numpy(x.astype(np.float32)).to(cuda).to(_tdt(dt))
    kv_write_q4(xt, xt, cache, torch.from_numpy(slots).to(cuda))
    want = qo.write(start, slots, x, x)
    np.testing.assert_array_equal(cache.cpu().numpy(), want)
    k, _ = kv_read_q4(cache, torch.from_numpy(slots).to(cuda), dtype=_tdt(dt))
    ref = po.round_to(qo.read(want, slots)[0], dt)
    np.testing.assert_array_equal(_host(k), ref)
    nan = np.isnan(ref[0, 0]).all(-1)
    assert nan[[0, 1, 2, 8]].all() and not np.isnan(ref[0, 0, [3, 4, 5, 6, 7, 9, 10, 11]]).any()


def test_empty_and_repeated_slots(cuda):
    import torch

    from kernelfoundry_b200 import kv_read_q4, kv_write_q4, q4_cache

    cache = q4_cache(2, 2, 16, 64, cuda)
    e = torch.empty(0, 2, 5, 64, device=cuda, dtype=torch.float16)
    es = torch.empty(0, 5, device=cuda, dtype=torch.int32)
    kv_write_q4(e, e, cache, es)
    assert kv_read_q4(cache, es)[0].shape == (0, 2, 5, 64) and (cache == 0).all()
    x = torch.randn(1, 2, 1, 64, device=cuda).half().expand(1, 2, 2, 64)   # one row for both tokens (stride 0)
    kv_write_q4(x, x, cache, torch.tensor([[7, 7]], dtype=torch.int32, device=cuda))
    k, v = kv_read_q4(cache, torch.tensor([[7, 8]], dtype=torch.int32, device=cuda))
    assert torch.equal(k, v) and (k[:, :, 0] - x[:, :, 0]).abs().max() < 0.3 and (k[:, :, 1] == 0).all()


def test_offsets_past_32_bits(cuda):
    """A pool over 4 GiB: the last block is written, read and attended."""
    import torch

    from kernelfoundry_b200 import flash_attn_paged_q4, kv_read_q4, kv_write_q4, q4_cache

    H, D, bs = 8, 128, 256
    n_blocks = (5 << 30) // (H * bs * (D + 8))
    cache = q4_cache(n_blocks, H, bs, D, cuda)
    assert cache.numel() > 1 << 32
    torch.manual_seed(2)
    k, v = (torch.randn(1, H, 40, D, device=cuda).half() for _ in range(2))
    slots = (torch.arange(40, device=cuda, dtype=torch.int32) + (n_blocks - 1) * bs)[None].contiguous()
    kv_write_q4(k, v, cache, slots)
    small = q4_cache(1, H, bs, D, cuda)
    ids = torch.arange(40, device=cuda, dtype=torch.int32)[None]
    kv_write_q4(k, v, small, ids)
    assert torch.equal(cache[-1], small[0]) and (cache[:-1].count_nonzero() == 0)
    a, b = kv_read_q4(cache, slots), kv_read_q4(small, ids)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    q = torch.randn(1, 32, 1, D, device=cuda).half()
    lens = torch.tensor([40], dtype=torch.int32, device=cuda)
    far = flash_attn_paged_q4(q, cache, torch.tensor([[n_blocks - 1]], dtype=torch.int32, device=cuda), lens)
    near = flash_attn_paged_q4(q, small, torch.tensor([[0]], dtype=torch.int32, device=cuda), lens)
    assert torch.equal(far, near)


# ------------------------------------------------------------------ attention
def _filled(rng, B, H, D, bs, lens, extra=1, poison=True):
    """A cache with every page's used slots written; unused slots and pages hold NaN scales and garbage codes."""
    per = max(1, max(-(-n // bs) for n in lens)) + extra
    n_blocks = B * per + 2
    cache = rng.integers(0, 256, (n_blocks, H, bs // 16, 16 * (D + 8)), dtype=np.uint8)
    words = cache[..., 16 * D:].view(np.uint32)
    words[...] = qo.BAD if poison else 0
    table = rng.permutation(n_blocks)[:B * per].reshape(B, per).astype(np.int32)
    for b, n in enumerate(lens):
        if n:
            j = np.arange(n)
            slots = (table[b, j // bs] * bs + j % bs)[None].astype(np.int32)
            gain = 1 + 3 * (rng.random((1, H, 1, D)) < 0.05)
            k, v = rng.standard_normal((1, H, n, D)) * gain, rng.standard_normal((1, H, n, D)) + 0.5
            cache = qo.write(cache, slots, k.astype(np.float16), v.astype(np.float16))
        table[b, -(-n // bs):] = 2 ** 30                 # never read
    return cache, table


def _attn(cuda, q, dt, cache, table, lens, **kw):
    import torch

    from kernelfoundry_b200 import flash_attn_paged_q4

    to = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(cuda)  # noqa: E731
    return flash_attn_paged_q4(_dev(q, dt, cuda), to(cache), to(table), to(np.asarray(lens, np.int32)), **kw)


def _check(got, ref, A, out_dt, what=""):
    got = _host(got)
    half_ulp = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}[out_dt]
    tol = 2.0 ** -10 * A + half_ulp * np.abs(ref) + (2.0 ** -25 if out_dt == "f16" else 0.0)
    bad = ~(np.abs(got - ref) <= tol)
    assert not bad.any(), f"{what}: {bad.sum()} outside, worst {np.nanmax(np.abs(got - ref) / np.maximum(tol, 1e-30)):.2f}x"


ATTN = [
    # H_q, H_kv, S_q, D, block_size, lens, causal, q dtype, out dtype
    (1, 1, 1, 64, 16, [1], False, "f16", "f16"),
    (8, 2, 1, 128, 16, [0, 1, 15, 16, 17, 31, 32, 33], False, "f16", "f16"),
    (32, 8, 1, 128, 16, [512], False, "f16", "f32"),
    (32, 8, 1, 128, 64, [700, 63, 64, 65, 0, 129], False, "bf16", "bf16"),
    (8, 8, 1, 64, 32, [47, 48, 300], False, "bf16", "f16"),
    (5, 1, 1, 256, 16, [100, 1, 777], False, "f16", "f16"),
    (7, 1, 1, 64, 128, [130, 260], False, "f16", "bf16"),
    (12, 4, 3, 128, 16, [1, 2, 3, 4, 40, 0], True, "f16", "f16"),
    (12, 4, 3, 128, 16, [1, 2, 3, 4, 40, 0], False, "f16", "f32"),
    (16, 4, 4, 128, 32, [65, 200], True, "bf16", "bf16"),
    (20, 4, 3, 256, 16, [3, 500, 33], True, "f16", "f16"),
    (32, 1, 2, 64, 256, [600, 5], True, "f16", "f32"),
    (16, 1, 4, 128, 16, [95, 4, 2], True, "bf16", "f32"),
    (6, 2, 5, 64, 16, [5, 6, 70, 16], True, "f16", "f16"),
    (64, 1, 1, 256, 64, [333], False, "f16", "f16"),
    (4, 4, 1, 128, 256, [255, 256, 257, 1000], False, "f16", "f16"),
]


@pytest.mark.parametrize("case", ATTN, ids=lambda c: "Hq{}_Hkv{}_Sq{}_D{}_bs{}_n{}_c{}_{}_{}".format(*c[:5], max(c[5]), *c[6:]))
def test_attention_matches_oracle(cuda, case):
    H_q, H_kv, S_q, D, bs, lens, causal, dt, out_dt = case
    rng = np.random.default_rng(H_q * 31 + D + bs + sum(lens))
    cache, table = _filled(rng, len(lens), H_kv, D, bs, lens)
    q = po.round_to(1.5 * rng.standard_normal((len(lens), H_q, S_q, D)), dt)
    O, Mi, Li, A = qo.attention(q, cache, table, lens, causal)
    got, mi, li = _attn(cuda, q, dt, cache, table, lens, causal=causal, out_dtype=_tdt(out_dt), return_lse=True)
    _check(got, O, A, out_dt)
    mi, li = _host(mi), _host(li)
    none = np.isinf(Mi)
    assert (mi[none] == -np.inf).all() and (li[none] == 0).all() and (_host(got)[none] == 0).all()
    assert (np.abs(mi - Mi)[~none] <= 2.0 ** -18 * np.maximum(np.abs(Mi[~none]), 1)).all()
    assert (np.abs(li - Li)[~none] <= 2.0 ** -12 * Li[~none]).all()


@pytest.mark.parametrize("shape", [(1, 8, 2, 20000, 128, 16), (2, 4, 1, 9000, 64, 256), (1, 16, 1, 5000, 256, 32)])
def test_long_contexts_are_split_and_merged(cuda, shape):
    B, H_q, H_kv, n, D, bs = shape
    rng = np.random.default_rng(n)
    lens = [n - 37 * b for b in range(B)]
    cache, table = _filled(rng, B, H_kv, D, bs, lens)
    q = po.round_to(rng.standard_normal((B, H_q, 1, D)), "f16")
    O, _, _, A = qo.attention(q, cache, table, lens)
    _check(_attn(cuda, q, "f16", cache, table, lens), O, A, "f16")


def test_many_short_sequences(cuda):
    """More sequences than SMs, lengths 0..60, so that most are finished by one warp and some cross CTAs."""
    rng = np.random.default_rng(9)
    lens = rng.integers(0, 61, 700).tolist()
    cache, table = _filled(rng, len(lens), 2, 64, 16, lens)
    q = po.round_to(rng.standard_normal((len(lens), 4, 1, 64)), "bf16")
    O, _, _, A = qo.attention(q, cache, table, lens)
    _check(_attn(cuda, q, "bf16", cache, table, lens), O, A, "bf16")


def test_mixed_lengths_with_one_dominant(cuda):
    rng = np.random.default_rng(10)
    lens = [3, 0, 6000, 1, 17, 0, 250]
    cache, table = _filled(rng, len(lens), 2, 128, 32, lens)
    q = po.round_to(rng.standard_normal((len(lens), 16, 2, 128)), "f16")
    O, _, _, A = qo.attention(q, cache, table, lens, causal=True)
    _check(_attn(cuda, q, "f16", cache, table, lens, causal=True), O, A, "f16")


@pytest.mark.parametrize("D,H_q,H_kv,n", [(64, 8, 2, 300), (128, 8, 1, 5000), (128, 16, 1, 700), (256, 4, 1, 900)])
def test_fp32_output_carries_more_than_fp16(cuda, D, H_q, H_kv, n):
    """With an fp32 output p goes in as two fp16 operands (2^-22 together); what is left are the scores' fp32 errors
    (absolute, below 2^-17 for these inputs, so as much relative in p) and the sums': 2^-16 A + 2^-24 |O|."""
    rng = np.random.default_rng(D + n)
    cache, table = _filled(rng, 1, H_kv, D, 16, [n])
    q = po.round_to(rng.standard_normal((1, H_q, 1, D)), "f16")
    O, _, _, A = qo.attention(q, cache, table, [n])
    got = _host(_attn(cuda, q, "f16", cache, table, [n], out_dtype=_tdt("f32")))
    tol = 2.0 ** -16 * A + 2.0 ** -24 * np.abs(O)
    assert (np.abs(got - O) <= tol).all(), f"worst {(np.abs(got - O) / tol).max():.2f}x"


def test_scale_growing_maximum_and_outlier_scales(cuda):
    """Scores that rise along the context (the running maximum moves in every tile), values whose scales span 2^40,
    an explicit softmax scale, a negative one."""
    rng = np.random.default_rng(11)
    n, H, D = 3000, 1, 128
    cache, table = _filled(rng, 1, H, D, 16, [n])
    j = np.arange(n)
    slots = (table[0, j // 16] * 16 + j % 16)[None].astype(np.int32)
    u = rng.standard_normal(D)
    k = np.linspace(0, 2, n)[:, None] * u + 0.1 * rng.standard_normal((n, D))
    v = rng.standard_normal((n, D)) * 2.0 ** rng.integers(-20, 20, (n, 1))
    cache = qo.write(cache, slots, k[None, None].astype(np.float32), v[None, None].astype(np.float32))
    q = po.round_to(np.stack([u, -u, 0 * u, rng.standard_normal(D)])[None, :, None], "bf16")
    for scale in (None, 0.31, -0.05):
        O, _, _, A = qo.attention(q, cache, table, [n], scale=scale)
        _check(_attn(cuda, q, "bf16", cache, table, [n], scale=scale, out_dtype=_tdt("f32")), O, A, "f32", f"scale {scale}")


def _with_rows(cache, table, bs, b, rows):
    """``cache`` with rows {key: (k or None, v or None)} of sequence b rewritten for every head (bf16 values, [D])."""
    H, D = cache.shape[1], cache.shape[-1] // 16 - 8
    for j, (k, v) in rows.items():
        t = int(table[b, j // bs] * bs + j % bs)
        old = [x[0, :, 0] for x in qo.read(cache, np.array([[t]]))]
        k, v = (po.round_to(np.broadcast_to(o if x is None else x, (H, D)), "bf16") for x, o in zip((k, v), old))
        cache = qo.write(cache, np.array([[t]], np.int32), k[None, :, None].astype(np.float32), v[None, :, None].astype(np.float32))
    return cache


def _check_rows(got, O, A, out_dt, what):
    """Outputs where one value row is far larger than the others.  p t (t: a value's scale) is rounded per key as
    elsewhere (within 2^-10 A), and by 2^-23 of the row's largest p t, as fp16 has a last bit.  The key with that
    largest one adds at least 7 times it to A in some dim, and a rounding moves an output by at most 15 times
    itself: 2^-21.9 max_d A a key, as many as 2^7 times that for 3000 independent ones: below 2^-13 max_d A."""
    got = _host(got)
    half_ulp = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}[out_dt]
    tol = 2.0 ** -10 * A + 2.0 ** -13 * A.max(-1, keepdims=True) + half_ulp * np.abs(O) + (2.0 ** -25 if out_dt == "f16" else 0.0)
    bad = ~(np.abs(got - O) <= tol)
    assert not bad.any(), f"{what}: {bad.sum()} outside, worst {np.nanmax(np.abs(got - O) / np.maximum(tol, 1e-30)):.2f}x"


@pytest.mark.parametrize("out_dt", ["bf16", "f32", "f16"])
@pytest.mark.parametrize("D,H_q,S_q", [(64, 4, 2), (64, 8, 2), (128, 4, 2), (128, 4, 4), (256, 2, 3)])
def test_a_huge_value_hidden_from_a_row_leaves_it_alone(cuda, D, H_q, S_q, out_dt):
    """The last draft's value is 1e20 (or 1e7): earlier drafts, which may not see it, are what they are without it."""
    rng = np.random.default_rng(40 + D + S_q)
    for n, big in ((40, 1e20), (40, 1e7), (3000, 1e20)):
        cache, table = _filled(rng, 1, 1, D, 16, [n])
        cache = _with_rows(cache, table, 16, 0, {n - 1: (None, np.full(D, big) * rng.uniform(0.5, 1, D))})
        q = po.round_to(rng.standard_normal((1, H_q, S_q, D)), "bf16")
        O, _, _, A = qo.attention(q, cache, table, [n], causal=True)
        got = _attn(cuda, q, "bf16", cache, table, [n], causal=True, out_dtype=_tdt(out_dt))
        if out_dt == "f16":                              # rows that see it are beyond fp16
            assert np.isinf(_host(got)[:, :, -1]).any() or big == 1e7
            got, O, A = got[:, :, :-1], O[:, :, :-1], A[:, :, :-1]
        _check_rows(got, O, A, out_dt, f"n {n}, value {big}")


@pytest.mark.parametrize("out_dt", ["bf16", "f32"])
@pytest.mark.parametrize("n", [30, 2000])
@pytest.mark.parametrize("at", ["first", "last"])
def test_a_huge_value_with_next_to_no_probability(cuda, n, at, out_dt):
    """One key scores 60 below the maximum and its value is 1e20: it adds about 1e-6, the others stay what they are."""
    D = 128
    rng = np.random.default_rng(50 + n)
    cache, table = _filled(rng, 1, 1, D, 16, [n])
    u = np.sign(rng.standard_normal(D))                  # scores: key . q / sqrt(D), q = u
    j = 0 if at == "first" else n - 1
    rows = {j: (-45 / np.sqrt(D) * u, np.full(D, 1e20) * rng.uniform(0.5, 1, D)), n // 2: (15 / np.sqrt(D) * u, None)}
    cache = _with_rows(cache, table, 16, 0, rows)
    q = po.round_to(np.stack([u, 0.5 * u, 0.25 * u, -0.1 * u])[None, :, None], "bf16")
    O, _, _, A = qo.attention(q, cache, table, [n])
    assert A[0, 0].max() < 100 < A[0, 3].max()           # negligible in the first row, everything in the last
    _check_rows(_attn(cuda, q, "bf16", cache, table, [n], out_dtype=_tdt(out_dt)), O, A, out_dt, at)


@pytest.mark.parametrize("out_dt", ["bf16", "f32"])
@pytest.mark.parametrize("tiny", [1.0, 1e-6, 1e-12])
@pytest.mark.parametrize("B,n", [(1500, 256), (1, 3000)])
def test_early_huge_values_outweighed_by_later_scores(cuda, B, n, tiny, out_dt):
    """Values of 1e15 lead while the scores are low; later keys outweigh the first of them by 2^115, with ordinary and with
    tiny values.  1500 sequences on the same pages give a warp whole units of 8 tiles, one sequence is split over all warps."""
    D, H = 128, 2
    rng = np.random.default_rng(60)
    cache, table = _filled(rng, 1, H, D, 16, [n])
    u = np.sign(rng.standard_normal(D))
    step = np.linspace(-40, 40, n)
    rows = {j: (step[j] / np.sqrt(D) * u, rng.standard_normal(D) * (1e15 if j < n // 4 else tiny)) for j in range(0, n, max(1, n // 256))}
    cache = _with_rows(cache, table, 16, 0, rows)
    q = po.round_to(np.stack([u, -u, 0.3 * u, 0 * u])[None, :, None], "bf16")
    O, _, _, A = qo.attention(q, cache, table, [n])
    got = _attn(cuda, np.repeat(q, B, 0), "bf16", cache, np.repeat(table, B, 0), [n] * B, out_dtype=_tdt(out_dt))
    _check_rows(got, O, A, out_dt, "")

def test_scores_of_any_size(cuda):
    """Scores near +-1e36 (bf16 queries and keys): equal keys weigh alike whatever the sign, a lower one nothing."""
    D = 64
    rng = np.random.default_rng(30)
    u = np.sign(rng.standard_normal(D))
    for n in (1, 20, 70):
        cache, table = _filled(rng, 1, 1, D, 16, [n])
        cache = _with_rows(cache, table, 16, 0, {j: (2.0 ** 55 * u * (0.5 if j == 13 else 1.0), None) for j in range(n)})
        q = po.round_to(np.stack([-u, u, 0.25 * u, -2.0 ** -100 * u])[None, :, None] * 2.0 ** 60, "bf16")
        O, Mi, Li, A = qo.attention(q, cache, table, [n])
        assert Mi.min() < -1e34 and Mi.max() > 1e34
        got, mi, li = _attn(cuda, q, "bf16", cache, table, [n], out_dtype=_tdt("f32"), return_lse=True)
        _check(got, O, A, "f32", f"n {n}")
        assert (np.abs(_host(mi) - Mi) <= 2.0 ** -18 * np.maximum(np.abs(Mi), 1)).all()
        assert (np.abs(_host(li) - Li) <= 2.0 ** -12 * Li).all()


@pytest.mark.parametrize("scale", [0.0, -0.0, 1e-60, 1e-30])
def test_a_scale_of_zero_is_not_the_default(cuda, scale):
    """scale=0 weighs all keys alike, and so does a scale too small for fp32; None is 1/sqrt(D)."""
    rng = np.random.default_rng(31)
    cache, table = _filled(rng, 2, 2, 128, 16, [75, 3])
    q = po.round_to(3 * rng.standard_normal((2, 8, 1, 128)), "f16")
    O, _, Li, A = qo.attention(q, cache, table, [75, 3], scale=scale)
    got, mi, li = _attn(cuda, q, "f16", cache, table, [75, 3], scale=scale, return_lse=True)
    _check(got, O, A, "f16")
    assert np.abs(_host(mi)).max() < 1e-25 and (np.abs(_host(li) - Li) <= 2.0 ** -12 * Li).all()


def test_query_magnitudes(cuda):
    """bf16 rows far apart in size (beyond fp16's range) in one call; a zero row attends uniformly."""
    rng = np.random.default_rng(12)
    lens = [90]
    cache, table = _filled(rng, 1, 1, 64, 16, lens)
    q = rng.standard_normal((1, 6, 1, 64)) * np.array([1e-20, 1e-3, 1.0, 1e4, 0.0, 1e6])[None, :, None, None]
    q = po.round_to(q, "bf16")
    for r in range(6):                                    # each row's scale keeps its scores of order one
        scale = 0.1 / max(np.abs(q[0, r]).max(), 1e-30)
        O, _, _, A = qo.attention(q[:, r:r + 1], cache, table, lens, scale=scale)
        got = _attn(cuda, q, "bf16", cache, table, lens, scale=scale)[:, r:r + 1]
        _check(got, O, A, "bf16", f"row {r}")


def test_bad_table_entries_read_zeros(cuda):
    rng = np.random.default_rng(13)
    for bs in (16, 64):
        lens = [150]
        cache, table = _filled(rng, 1, 2, 128, bs, lens)
        table[0, 1] = -1
        if bs == 16:
            table[0, 4] = 2 ** 30
        q = po.round_to(rng.standard_normal((1, 8, 1, 128)), "f16")
        O, _, _, A = qo.attention(q, cache, table, lens)
        _check(_attn(cuda, q, "f16", cache, table, lens), O, A, "f16")


def test_poisoned_rows_reach_only_those_that_see_them(cuda):
    """A key with a NaN: queries before it (causal) stay clean, later ones are NaN; other sequences and heads are clean."""
    rng = np.random.default_rng(14)
    lens = [40, 40]
    cache, table = _filled(rng, 2, 2, 128, 16, lens)
    bad = rng.standard_normal((1, 1, 1, 128))
    bad[..., 7] = np.nan
    t = table[0, 39 // 16] * 16 + 39 % 16                # the last key of sequence 0 ...
    clean = cache.copy()
    x = qo.write(cache, np.array([[t]], np.int32), np.broadcast_to(bad, (1, 2, 1, 128)), np.broadcast_to(bad, (1, 2, 1, 128)))
    cache[t // 16, 0] = x[t // 16, 0]                    # ... of head 0 only
    q = po.round_to(rng.standard_normal((2, 4, 3, 128)), "f16")
    got = _host(_attn(cuda, q, "f16", cache, table, lens, causal=True))
    O, _, _, A = qo.attention(q, clean, table, lens, causal=True)
    assert np.isnan(got[0, :2, 2]).all()
    got[0, :2, 2], O[0, :2, 2] = 0, 0
    assert np.isfinite(got).all()
    import torch

    _check(torch.from_numpy(got), O, A, "f16")


def test_lengths_are_clamped_and_negative_is_empty(cuda):
    rng = np.random.default_rng(15)
    cache, table = _filled(rng, 3, 1, 64, 16, [32, 32, 32], extra=0, poison=False)
    q = po.round_to(rng.standard_normal((3, 2, 1, 64)), "f16")
    lens = [32, 1000, -5]
    O, _, _, A = qo.attention(q, cache, table, lens)
    got = _attn(cuda, q, "f16", cache, table, lens)
    _check(got, O, A, "f16")
    assert (got[2] == 0).all()


def test_repeatable_streams_graphs_and_shared_workspace(cuda):
    """Bit-equal results: twice in a row, on another stream, from a captured graph with new lengths, and after the
    fp16 paged decode used the same workspace."""
    import torch

    from kernelfoundry_b200 import flash_attn_paged_q4
    from kernelfoundry_b200._lib import lib
    from kernelfoundry_b200.attention import device_error, flash_attn_paged, new_workspace

    rng = np.random.default_rng(16)
    lens = [3000, 10, 1234]
    cache, table = _filled(rng, 3, 2, 128, 16, lens, poison=False)
    to = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(cuda)  # noqa: E731
    q, c, t, n = _dev(rng.standard_normal((3, 8, 1, 128)), "f16", cuda), to(cache), to(table), to(np.array(lens, np.int32))
    t.clamp_(0, cache.shape[0] - 1)
    a = flash_attn_paged_q4(q, c, t, n)
    for _ in range(3):
        assert torch.equal(flash_attn_paged_q4(q, c, t, n), a)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        b = flash_attn_paged_q4(q, c, t, n)
    side.synchronize()
    assert torch.equal(a, b)
    need = lib().kf_attn_paged_q4_workspace_bytes(3, 8, 2, 1, 128, 16, t.shape[1])
    ws = new_workspace(max(need, lib().kf_attn_paged_workspace_bytes(3, 8, 2, 1, 128, 16, t.shape[1])), cuda)
    pool = torch.randn(cache.shape[0], 2, 16, 128, device=cuda).half()
    first = flash_attn_paged(q, pool, pool, t, n, workspace=ws)
    assert torch.equal(flash_attn_paged_q4(q, c, t, n, workspace=ws), a)
    assert torch.equal(flash_attn_paged(q, pool, pool, t, n, workspace=ws), first)
    out = torch.empty_like(a)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        flash_attn_paged_q4(q, c, t, n, out=out, workspace=ws)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, a)
    n.copy_(to(np.array([17, 3001, 0], np.int32)))       # the lengths live on the device
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, flash_attn_paged_q4(q, c, t, n))
    assert device_error()[0] == 0


def test_graph_keeps_its_streams_workspace(cuda):
    """A graph captured with the stream's own workspace stays right after calls that need a larger one and new tensors
    that could have taken its place."""
    import torch

    from kernelfoundry_b200 import flash_attn_paged_q4

    rng = np.random.default_rng(23)
    to = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(cuda)  # noqa: E731
    inputs = []
    for D, H_q in ((64, 4), (128, 32), (256, 4)):
        cache, table = _filled(rng, 2, 2, D, 16, [700, 90], poison=False)
        t = to(table).clamp_(0, cache.shape[0] - 1)
        inputs.append((_dev(rng.standard_normal((2, H_q, 1, D)), "f16", cuda), to(cache), t, to(np.array([700, 90], np.int32))))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        want = flash_attn_paged_q4(*inputs[0])
        out = torch.empty_like(want)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            flash_attn_paged_q4(*inputs[0], out=out)
        others = [flash_attn_paged_q4(*x) for x in inputs[1:]]
        junk = [torch.full((n,), 255, dtype=torch.uint8, device=cuda) for n in (1 << 19, 1 << 20, 1 << 21, 1 << 21)]
        graph.replay()
        stream.synchronize()
        assert torch.equal(out, want)
        assert all(bool((j == 255).all()) for j in junk)
        assert all(torch.equal(flash_attn_paged_q4(*x), y) for x, y in zip(inputs[1:], others))
        stream.synchronize()


def test_written_cache_attends_like_its_read_back_values(cuda):
    """write -> attend equals read back -> flash_attn_fwd within both calls' rounding (K, V rounded to fp16 on read)."""
    import torch

    from kernelfoundry_b200 import flash_attn_fwd, flash_attn_paged_q4, kv_read_q4, kv_write_q4, q4_cache

    torch.manual_seed(4)
    B, H_q, H_kv, n, D, bs = 2, 32, 8, 512, 128, 16
    cache = q4_cache(B * n // bs, H_kv, bs, D, cuda)
    table = torch.randperm(B * n // bs, device=cuda).int().view(B, -1)
    slots = (table[:, :, None] * bs + torch.arange(bs, device=cuda, dtype=torch.int32)).view(B, n).contiguous()
    k, v = (torch.randn(B, H_kv, n, D, device=cuda).half() for _ in range(2))
    kv_write_q4(k, v, cache, slots)
    q = torch.randn(B, H_q, 1, D, device=cuda).half()
    a = flash_attn_paged_q4(q, cache, table, torch.full((B,), n, dtype=torch.int32, device=cuda), out_dtype=torch.float32)
    kr, vr = kv_read_q4(cache, slots)
    b = flash_attn_fwd(q, kr, vr)
    assert (a - b).abs().max() < 4e-3


def test_refusals(cuda):
    import torch

    from kernelfoundry_b200 import KFError, flash_attn_paged_q4, kv_read_q4, kv_write_q4, q4_cache

    for bad in ((4, 2, 24, 128), (4, 2, 8, 128), (4, 2, 16, 96), (4, 2, 512, 128)):
        with pytest.raises(ValueError):
            q4_cache(*bad, cuda)
    c = q4_cache(4, 2, 16, 128, cuda)
    k = torch.zeros(1, 2, 8, 128, device=cuda, dtype=torch.float16)
    s = torch.zeros(1, 8, device=cuda, dtype=torch.int32)
    for args in ((k.cpu(), k, c, s), (k, k.bfloat16(), c, s), (k, k[:, :, :4], c, s), (k[:, :1], k[:, :1], c, s),
                 (k, k, c, s.long()), (k, k, c, s[:, :4]), (k, k, c.cpu(), s), (k, k, c.view(torch.int32), s),
                 (k, k, c[..., :-16], s), (k.float(), k.float(), c, s)):
        with pytest.raises(ValueError):
            kv_write_q4(*args)
    with pytest.raises(ValueError):
        kv_write_q4(k, k, c, s, layout="hbsd")
    odd = torch.zeros(8 * 256 + 4, device=cuda, dtype=torch.float16)[4:].view(1, 2, 8, 128)
    with pytest.raises(KFError, match="aligned"):
        kv_write_q4(odd, k, c, s)
    for kw in (dict(dtype=torch.float32), dict(layout="x"), dict(out=(k, k[:, :1]))):
        with pytest.raises(ValueError):
            kv_read_q4(c, s, **kw)
    q = torch.zeros(1, 4, 1, 128, device=cuda, dtype=torch.float16)
    t = torch.zeros(1, 4, device=cuda, dtype=torch.int32)
    n = torch.full((1,), 5, device=cuda, dtype=torch.int32)
    for args, kw in (((q.float(), c, t, n), {}), ((q[..., :64], c, t, n), {}), ((q, c, t.long(), n), {}), ((q, c, t, n.long()), {}),
                     ((q, c, t, n[:0]), {}), ((q, c, t, n), dict(out_dtype=torch.float64)),
                     ((q, c, t, n), dict(out=torch.zeros(1, 4, 1, 64, device=cuda))), ((q.transpose(1, 2), c, t, n.cpu()), {})):
        with pytest.raises(ValueError):
            flash_attn_paged_q4(*args, **kw)
    with pytest.raises(KFError, match="invalid"):
        flash_attn_paged_q4(torch.zeros(1, 3, 1, 128, device=cuda, dtype=torch.float16), c, t, n)     # 3 % 2
    with pytest.raises(KFError, match="invalid"):
        flash_attn_paged_q4(torch.zeros(1, 4, 40, 128, device=cuda, dtype=torch.float16), c, t, n)    # 80 rows a cache head
    with pytest.raises(KFError, match="invalid"):
        flash_attn_paged_q4(q, c, t, n, scale=float("nan"))
    e = torch.zeros(0, 4, 1, 128, device=cuda, dtype=torch.float16)
    assert flash_attn_paged_q4(e, c, t[:0], n[:0]).shape == e.shape


def test_refused_workspaces(cuda):
    """Refused on the host, also once a call of the same form has gone through; a good one still does."""
    import torch

    from kernelfoundry_b200 import KFError, flash_attn_paged_q4, q4_cache
    from kernelfoundry_b200.attention import new_workspace

    q = torch.zeros(1, 4, 1, 128, device=cuda, dtype=torch.float16)
    args = (q, q4_cache(4, 2, 16, 128, cuda), torch.zeros(1, 4, device=cuda, dtype=torch.int32),
            torch.full((1,), 5, device=cuda, dtype=torch.int32))
    n = 1 << 22
    good = new_workspace(n, cuda)
    want = flash_attn_paged_q4(*args, workspace=good)
    for bad in (torch.zeros(n, dtype=torch.uint8), torch.zeros(n, dtype=torch.uint8).pin_memory(),
                torch.zeros(n, device=cuda), torch.zeros(2 * n, dtype=torch.uint8, device=cuda)[::2]):
        with pytest.raises(ValueError, match="workspace"):
            flash_attn_paged_q4(*args, workspace=bad)
    with pytest.raises(KFError):
        flash_attn_paged_q4(*args, workspace=good[:1024])
    assert torch.equal(flash_attn_paged_q4(*args, workspace=good), want)


# ------------------------------------------------------------------ sizes at which a thread or a warp goes on to the next
LARGE_IO = [
    # B, S, H, D, block_size, dtype: rows for two passes of a write's block and four of a read's
    (1, 5431, 7, 128, 16, "f16"),
    (3, 1700, 8, 128, 64, "bf16"),
    (2, 9503, 4, 64, 32, "bf16"),
    (1, 2413, 8, 256, 128, "f16"),
]


@pytest.mark.parametrize("case", LARGE_IO, ids=lambda c: "B{}_S{}_H{}_D{}_bs{}_{}".format(*c))
@pytest.mark.parametrize("layout", ["bhsd", "bshd"])
def test_write_and_read_of_several_passes(cuda, case, layout):
    B, S, H, D = case[:4]
    assert B * S * 2 * H >= 4 * (4096 // D) * 4 * 148    # where both launchers begin to give a block all its passes
    test_write_bytes_and_read_values(cuda, case, layout)


def _alternating(cuda, rng, cache, table, B, H_q, S_q, D, lens, dt, out_dt, causal, check):
    """B sequences on the pages of one: lengths and queries alternate between two, results against the oracle for all."""
    q = po.round_to(rng.standard_normal((2, H_q, S_q, D)), dt)
    O, _, _, A = qo.attention(q, cache, np.repeat(table, 2, 0), lens, causal)
    pick = np.arange(B) % 2
    got = _attn(cuda, q[pick], dt, cache, np.repeat(table, B, 0), np.array(lens)[pick], causal=causal, out_dtype=_tdt(out_dt))
    check(got, O[pick], A[pick], out_dt, "")


@pytest.mark.parametrize("D,H_q,S_q,B,dt,out_dt", [(128, 8, 1, 64, "f16", "f16"), (128, 5, 1, 64, "bf16", "bf16"), (64, 4, 1, 84, "f16", "f32"),
                                                   (64, 2, 8, 64, "f16", "f16"), (128, 4, 4, 44, "f16", "f16"), (128, 4, 3, 44, "bf16", "bf16"),
                                                   (256, 4, 2, 44, "f16", "f16"), (256, 1, 1, 44, "bf16", "bf16")])
@pytest.mark.parametrize("bs", [16, 128])
def test_warps_with_more_than_a_window_of_tiles(cuda, D, H_q, S_q, B, dt, out_dt, bs):
    """Shares of 33 tiles and more for every warp: each ring stage is filled many times, the window of 32 tiles moves on,
    and the maximum (by 58 bits) and the values' scales (by 2^20) grow again and again inside a share."""
    rng = np.random.default_rng(D + 10 * H_q + S_q + bs)
    n = 32000
    warps = {(64, False): 16, (64, True): 12, (128, False): 12, (128, True): 8, (256, False): 8, (256, True): 8}[D, H_q * S_q > 8]
    assert B * (n // 32) * (2 if D == 256 and H_q * S_q > 8 else 1) >= 33 * warps * 148
    cache, table = _filled(rng, 1, 1, D, bs, [n])
    _alternating(cuda, rng, cache, table, B, H_q, S_q, D, [n, n - 37], dt, out_dt, S_q > 1, _check)
    u = np.sign(rng.standard_normal(D))
    j = np.arange(n)
    k = (40 / np.sqrt(D)) * (j % 1000 / 1000)[:, None] * u + 0.1 * rng.standard_normal((n, D))
    v = rng.standard_normal((n, D)) * 2.0 ** np.floor(20 * (j % 700 / 700) - 15)[:, None]
    slots = (table[0, j // bs] * bs + j % bs)[None].astype(np.int32)
    cache = qo.write(cache, slots, k[None, None].astype(np.float32), v[None, None].astype(np.float32))
    q = po.round_to(np.stack([np.broadcast_to(f * u, (H_q, S_q, D)) for f in (1.0, 0.5)]), dt)
    O, _, _, A = qo.attention(q, cache, np.repeat(table, 2, 0), [n, n - 37], S_q > 1)
    pick = np.arange(B) % 2
    got = _attn(cuda, q[pick], dt, cache, np.repeat(table, B, 0), np.array([n, n - 37])[pick], causal=S_q > 1, out_dtype=_tdt(out_dt))
    _check_rows(got, O[pick], A[pick], out_dt, "growing")


@pytest.mark.parametrize("D,H_q,S_q", [(64, 8, 1), (128, 8, 1), (128, 4, 4), (256, 8, 1)])
def test_full_batches_of_equal_lengths(cuda, D, H_q, S_q):
    """64 sequences of 4096 keys with 8 cache heads: whole units and units cut between CTAs, several to a warp's share."""
    rng = np.random.default_rng(D + S_q)
    H, n = 8, 4096
    cache, table = _filled(rng, 1, H, D, 16, [n])
    _alternating(cuda, rng, cache, table, 64, H_q * H, S_q, D, [n, n], "f16", "f16", S_q > 1, _check)
