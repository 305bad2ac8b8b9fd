"""Refusals of codebook_lookup, from the Python entry point and from the C ABI, without a GPU."""

import ctypes

import pytest
import torch

import gswarp_b200 as gs
from gswarp_b200 import _lib, codebook

T = torch.zeros(4, 3)
C = torch.zeros(5, dtype=torch.int64)


@pytest.mark.parametrize("args, message", [
    ((None, C), "torch.Tensor"),
    ((T, [0, 1]), "torch.Tensor"),
    ((torch.zeros(4), C), "at least two dimensions"),
    ((T.double(), C), "float32, bfloat16 or float16"),
    ((T.int(), C), "float32, bfloat16 or float16"),
    ((T, C.float()), "int32 or int64"),
    ((T, C.to(torch.int16)), "int32 or int64"),
    ((T, C), "same CUDA device"),
])
def test_bad_arguments_are_value_errors(args, message):
    with pytest.raises(ValueError, match=message):
        gs.codebook_lookup(*args)


@pytest.mark.parametrize("table, codes, scale, message", [
    ((4, 0), (5,), 1.0, "elements"),
    ((4, (1 << 22) + 1), (5,), 1.0, "elements"),
    (((1 << 31) - 1, 1), (5,), 1.0, "rows"),
    ((4, 3), ((1 << 31) - 4096,), 1.0, "rows"),
    ((4, 3), (5,), "2", "number"),
    ((4, 3), (5,), True, "number"),
    ((4, 3), (5,), torch.ones(4), "scale tensor"),
    ((4, 3), (5,), torch.ones(5, dtype=torch.float64), "scale tensor"),
])
def test_bad_sizes_and_scales(monkeypatch, table, codes, scale, message):
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda self: True))
    t = torch.empty(table, device="meta")
    c = torch.empty(codes, dtype=torch.int64, device="meta")
    if isinstance(scale, torch.Tensor):
        scale = scale.to("meta")
    with pytest.raises(ValueError, match=message):
        codebook._validate(t, c, scale)


def _args(**kw):
    a = _lib.CodebookArgs()
    a.P, a.K, a.D = 10, 4, 3
    a.scale = 1.0
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw", [dict(P=-1), dict(P=(1 << 31) - 4096), dict(K=-1), dict(K=(1 << 31) - 1), dict(D=0),
                                dict(D=(1 << 22) + 1), dict(dtype=3), dict(dtype=-1), dict()])
def test_c_abi_refuses(kw):
    L = _lib.load()
    for fn in (L.gsb_codebook_fwd, L.gsb_codebook_bwd):
        assert fn(ctypes.byref(_args(**kw)), None) == _lib.GSB_ERR_INVALID
        assert b"gsb_codebook" in L.gsb_last_error()


def test_c_abi_refuses_missing_buffers():
    L = _lib.load()
    p = 256  # any non-null address: every call below is refused before a launch
    full = dict(codes=p, table=p, error_word=p)
    assert L.gsb_codebook_fwd(ctypes.byref(_args(**full)), None) == _lib.GSB_ERR_INVALID  # no out
    assert L.gsb_codebook_bwd(ctypes.byref(_args(**full)), None) == _lib.GSB_ERR_INVALID  # no grad_out
    full["grad_out"] = p
    assert L.gsb_codebook_bwd(ctypes.byref(_args(grad_gain=p, **full)), None) == _lib.GSB_ERR_INVALID  # no gain
    bare = {**full, "table": None, "out": p, "gain": p}
    assert L.gsb_codebook_bwd(ctypes.byref(_args(grad_gain=p, **bare)), None) == _lib.GSB_ERR_INVALID  # no table
    assert L.gsb_codebook_fwd(ctypes.byref(_args(**bare)), None) == _lib.GSB_ERR_INVALID
    need = L.gsb_codebook_bwd_workspace_bytes(100_000, 400, 3)
    assert need > 0
    short = _args(P=100_000, K=400, grad_table=p, workspace=p, workspace_bytes=need - 1, **full)
    assert L.gsb_codebook_bwd(ctypes.byref(short), None) == _lib.GSB_ERR_INVALID
    assert L.gsb_codebook_fwd(None, None) == _lib.GSB_ERR_INVALID


def test_workspace_grows_with_the_rows_and_their_width():
    ws = _lib.load().gsb_codebook_bwd_workspace_bytes
    assert ws(0, 4, 3) == 0 and ws(10_000, 256, 3) == 0  # few rows need none
    assert ws(1_000_000, 4096, 45) >= 16 * 1_000_000
    assert ws(2_000_000, 4096, 45) > ws(1_000_000, 4096, 45)
    assert ws(1_000_000, 4096, 96) > ws(1_000_000, 4096, 45)


@pytest.mark.parametrize("sh, codes, message", [
    (torch.empty(4, 1, 3, device="meta"), torch.zeros(7, dtype=torch.int64), "sh codebook must be on cpu"),
    (torch.zeros(4, 1, 3), [0] * 7, "sh_codes must be"),
    (torch.zeros(4, 1, 3), torch.zeros(7, dtype=torch.int64, device="meta"), "sh_codes must be"),
])
def test_fused_step_refuses_codebooks_and_codes_elsewhere(sh, codes, message):
    from gswarp_b200.training import FusedViewStep

    params = [torch.zeros(7, n) for n in (3, 3, 4, 1)] + [sh]
    with pytest.raises(ValueError, match=message):
        FusedViewStep(params, ["a view"], sh_codes=codes)
