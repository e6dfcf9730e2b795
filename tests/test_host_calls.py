"""_kf_host.so, the host side of the small operators' Python calls (csrc/kf_host.cpp), without a GPU."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def host(kf_lib):
    from kernelfoundry_b200._lib import host

    return host()


def test_form_tells_apart_what_a_calls_checks_depend_on(host):
    a = torch.empty(2, 3, 4, dtype=torch.float16)
    same = [torch.empty(2, 3, 4, dtype=torch.float16), torch.ones(5, 3, 4, dtype=torch.float16)[1:3]]
    other = [a.to(torch.bfloat16), a.transpose(0, 1), torch.empty(2, 3, 8, dtype=torch.float16)[..., :4], a[0],
             torch.empty(2, 3, 5, dtype=torch.float16), a.reshape(2, 3, 4, 1), torch.empty(2, 3, 4, dtype=torch.float16, device="meta"), None]
    assert all(host.form(a) == host.form(t) for t in same)
    forms = [host.form(t) for t in [a, *other]]
    assert len(set(forms)) == len(forms)
    assert host.form(a, None) != host.form(None, a) != host.form(None, None, a)
    assert host.form() == b""
    assert host.form(torch.tensor(1.0), a) != host.form(a, torch.tensor(1.0))


def test_refusals(host):
    t = torch.zeros(1)
    for bad in (1, "x", [1.0], b"t"):
        with pytest.raises(TypeError, match="torch.Tensor"):
            host.form(t, bad)
    for call, n in ((host.kv_io, 6), (host.attn_q4, 11), (host.qk_norm_rope, 13)):
        with pytest.raises(TypeError, match=f"{n} arguments"):
            call(b"")
        with pytest.raises(ValueError, match="plan"):
            call(b"\0" * 8, *[None] * (n - 1))
        with pytest.raises(TypeError):
            call(None, *[None] * (n - 1))


def test_calls_reach_the_c_functions_with_their_arguments(host, kf_lib):
    """The C functions' own refusals come back as statuses: sizes, strides and flags are where they belong."""
    from kernelfoundry_b200 import _lib

    t = torch.zeros(64, dtype=torch.uint8)
    io = lambda dims, flags=0, st=(64, 64, 64) * 2: _lib.host_plan(kf_lib.kf_kv_write_q4, st, dims, flags)  # noqa: E731
    assert host.kv_io(io((1, 0, 1, 128, 1, 16)), t, t, t, t, 0) == _lib.KF_OK                       # no token: nothing to do
    assert host.kv_io(io((1, 1, 1, 96, 1, 16)), t, t, t, t, 0) == _lib.KF_ERR_UNSUPPORTED_HEAD_DIM
    assert host.kv_io(io((1, 1, 1, 128, 1, 24)), t, t, t, t, 0) == _lib.KF_ERR_INVALID_ARG
    assert host.kv_io(io((1, 0, 1, 128, 1, 16), flags=2), t, t, t, t, 0) == _lib.KF_ERR_INVALID_ARG
    assert host.kv_io(io((2, 2, 2, 128, 1, 16), st=(64, 64, 64, 64, 64, 60)), t, t, t, t, 0) == _lib.KF_ERR_INVALID_ARG
    attn = lambda dims, flags=0: _lib.host_plan(kf_lib.kf_attn_fwd_paged_q4, (), dims, flags)  # noqa: E731
    rest = (t, t, t, t, t, None, None, 0.0, t, 0)
    assert host.attn_q4(attn((0, 8, 2, 1, 128, 1, 16, 1)), *rest) == _lib.KF_OK
    assert host.attn_q4(attn((1, 8, 2, 1, 80, 1, 16, 1)), *rest) == _lib.KF_ERR_UNSUPPORTED_HEAD_DIM
    assert host.attn_q4(attn((1, 8, 3, 1, 128, 1, 16, 1)), *rest) == _lib.KF_ERR_INVALID_ARG
    assert host.attn_q4(attn((0, 8, 2, 1, 128, 1, 16, 1)), *rest[:7], float("inf"), t, 0) == _lib.KF_ERR_INVALID_ARG
    rope = lambda dims, st=(64,) * 12: _lib.host_plan(kf_lib.kf_qk_norm_rope, st, dims, 0)  # noqa: E731
    rest = (t, t, None, None, t, t, None, None)
    assert host.qk_norm_rope(rope((1, 0, 2, 1, 64, 64)), *rest, 1e4, 1.0, 1e-6, 0) == _lib.KF_OK
    assert host.qk_norm_rope(rope((1, 0, 2, 1, 64, 64)), *rest, 1e4, 1.0, -1.0, 0) == _lib.KF_ERR_INVALID_ARG
    assert host.qk_norm_rope(rope((1, 0, 2, 1, 64, 64)), *rest, -1.0, 1.0, 1e-6, 0) == _lib.KF_ERR_INVALID_ARG
    assert host.qk_norm_rope(rope((2, 2, 2, 1, 64, 64), st=(64,) * 11 + (60,)), *rest, 1e4, 1.0, 1e-6, 0) == _lib.KF_ERR_INVALID_ARG


def test_plan_sizes_are_the_structs(host):
    from kernelfoundry_b200 import _lib

    fn = ctypes.CFUNCTYPE(ctypes.c_int)(lambda: 0)
    assert len(_lib.host_plan(fn, range(6), range(6), 0)) == 88
    assert len(_lib.host_plan(fn, (), range(8), 0)) == 48
    assert len(_lib.host_plan(fn, range(12), range(6), 0)) == 136
    with pytest.raises(Exception, match="format|range"):
        _lib.host_plan(fn, range(6), (1 << 31,) * 6, 0)
