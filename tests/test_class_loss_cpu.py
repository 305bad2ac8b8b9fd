"""Refusals of class_cross_entropy, from the Python entry point and from the C ABI, without a GPU."""

import ctypes

import pytest
import torch

import gswarp_b200 as gs
from gswarp_b200 import _lib, class_loss

X, W, Y = torch.zeros(6, 4), torch.zeros(5, 4), torch.zeros(6, dtype=torch.int64)


def meta(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("args, kw, message", [
    ((None, W, Y), {}, "torch.Tensor"),
    ((X, W, [0] * 6), {}, "torch.Tensor"),
    ((torch.zeros(6), W, Y), {}, "shape"),
    ((torch.zeros(1, 1, 1, 1, 1), W, Y), {}, "shape"),
    ((X, W, Y[:5]), {}, "labels must have shape"),
    ((torch.zeros(2, 4, 3, 5), W, torch.zeros(2, 5, 3, dtype=torch.int64)), {}, "labels must have shape"),
    ((X, torch.zeros(5, 3), Y), {}, "weight must have shape"),
    ((X, torch.zeros(0, 4), Y), {}, "weight must have shape"),
    ((X, W.half(), Y), {}, "one dtype"),
    ((X.double(), W.double(), Y), {}, "one dtype"),
    ((X, W, Y.float()), {}, "int32 or int64"),
    ((torch.zeros(6, 129), torch.zeros(5, 129), Y), {}, "1 to 128 channels"),
    ((torch.zeros(6, 257).half(), torch.zeros(5, 257).half(), Y), {}, "1 to 256 channels"),
    ((torch.zeros(6, 0), torch.zeros(5, 0), Y), {}, "channels"),
    ((X, W, Y), dict(bias=torch.zeros(4)), "bias"),
    ((X, W, Y), dict(bias=torch.zeros(5).half()), "bias"),
    ((X, W, Y), {}, "same CUDA device"),
    ((meta((1 << 31) - 128, 1), meta(2, 1), meta((1 << 31) - 128, dtype=torch.int64)), {}, "fewer than"),
    ((meta(4, 1), meta((1 << 31) - 128, 1), meta(4, dtype=torch.int64)), {}, "fewer than"),
])
def test_bad_arguments_are_value_errors(args, kw, message):
    with pytest.raises(ValueError, match=message):
        gs.class_cross_entropy(*args, **kw)


@pytest.mark.parametrize("kw, message", [
    (dict(ignore_index=1.0), "ignore_index"), (dict(ignore_index=True), "ignore_index"),
    (dict(ignore_index=1 << 63), "64 bits"), (dict(reduction="avg"), "reduction"), (dict(train=1), "train"),
])
def test_bad_options(monkeypatch, kw, message):
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda self: True))
    with pytest.raises(ValueError, match=message):
        gs.class_cross_entropy(X, W, Y, **kw)


@pytest.mark.parametrize("shape, strides, copied", [
    ((6, 4), (4, 1), False), ((6, 4), (9, 1), False), ((6, 4), (1, 6), True), ((6, 1), (3, 7), False),
    ((4, 3, 5), (15, 5, 1), False), ((4, 3, 5), (40, 10, 2), False), ((4, 3, 5), (100, 8, 1), True),
    ((2, 4, 3, 5), (60, 15, 5, 1), False), ((2, 4, 3, 5), (60, 1, 20, 4), True), ((2, 1, 3, 5), (15, 1, 5, 1), False),
    ((2, 4, 1, 5), (60, 15, 99, 1), False), ((2, 4, 3, 1), (60, 15, 5, 1), True), ((2, 4, 3, 5), (0, 15, 5, 1), False),
])
def test_rows_address_every_element_of_a_strided_map(shape, strides, copied):
    size = 1 + sum((n - 1) * s for n, s in zip(shape, strides))
    x = torch.arange(float(size)).as_strided(shape, strides)
    y, B, S, C, (sb, sc, ss) = class_loss._rows(x)
    assert (y.data_ptr() != x.data_ptr()) == copied
    assert (sc == 1) == (x.ndim == 2)  # what the kernels tell the two gradient layouts apart by
    flat = y.as_strided((y.untyped_storage().nbytes() // 4,), (1,))
    n, c = torch.arange(B * S)[:, None], torch.arange(C)[None]
    got = flat[n // S * sb + c * (sc if C > 1 else 0) + n % S * ss]
    want = x if x.ndim == 2 else (x[None] if x.ndim == 3 else x).permute(0, 2, 3, 1).reshape(B * S, C)
    assert torch.equal(got, want)


def _args(**kw):
    a = _lib.ClassLossArgs()
    a.B, a.S, a.V, a.C, a.reduction, a.train = 1, 10, 4, 3, 2, 1
    for k in ("kept", "error_word", "workspace", "features", "weight", "labels", "loss", "upstream"):
        setattr(a, k, 256)  # refused before anything reads them
    a.workspace_bytes = 1 << 40
    for k, v in kw.items():
        setattr(a, k, v)
    return a


SIZES = [dict(B=-1), dict(S=-1), dict(S=(1 << 31) - 128), dict(B=1 << 20, S=1 << 20), dict(B=1 << 31), dict(V=0),
         dict(V=(1 << 31) - 128), dict(C=0), dict(C=129), dict(C=257, dtype=1), dict(dtype=3), dict(reduction=3)]
BUFFERS = [dict(kept=None), dict(workspace=None), dict(error_word=None), dict(workspace_bytes=0), dict(kept=264),
           dict(workspace=264)]


@pytest.mark.parametrize("kw", SIZES + BUFFERS)
def test_c_abi_refuses(kw):
    L = _lib.load()
    for fn in (L.gsb_class_loss_fwd, L.gsb_class_loss_bwd):
        assert fn(ctypes.byref(_args(**kw)), None) == _lib.GSB_ERR_INVALID
        assert b"gsb_class_loss" in L.gsb_last_error()


def test_c_abi_refuses_missing_inputs():
    L = _lib.load()
    for k in ("features", "weight", "labels", "loss"):
        assert L.gsb_class_loss_fwd(ctypes.byref(_args(**{k: None})), None) == _lib.GSB_ERR_INVALID
    assert L.gsb_class_loss_bwd(ctypes.byref(_args(upstream=None)), None) == _lib.GSB_ERR_INVALID
    assert L.gsb_class_loss_bwd(ctypes.byref(_args(train=0)), None) == _lib.GSB_ERR_INVALID
    assert L.gsb_class_loss_fwd(None, None) == _lib.GSB_ERR_INVALID


def _sizes(**kw):
    out = (ctypes.c_size_t * 3)()
    status = _lib.load().gsb_class_loss_sizes(ctypes.byref(_args(**kw)), out)
    return status, list(out)


def test_buffer_sizes():
    for kw in SIZES:
        assert _sizes(**kw)[0] == _lib.GSB_ERR_INVALID
    # the packed operands: planes of bf16, channels to a multiple of 16, rows and classes to 128
    status, (kept, fwd, bwd) = _sizes(S=129, V=300, C=17, dtype=0)
    packed = 3 * 32 * 2 * (256 + 384)
    assert status == _lib.GSB_OK and packed <= kept <= packed + 4 * (384 + 2 * 256) + 6 * 256
    assert fwd > 0 and bwd > 0
    assert _sizes(S=1_000_000)[1][0] > _sizes()[1][0]
    assert _sizes(S=0)[0] == _lib.GSB_OK
