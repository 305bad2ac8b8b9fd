"""class_cross_entropy against its definition in 64 bits.

The tolerance of every output is a bound counted from the roundings, with
u = 2^-24 and sums of magnitudes in place of sums:

* a logit: every product is exact to 2 u (three bf16 planes hold an fp32
  value to u, dropped cross products are below u; 16-bit inputs are exact),
  and each of at most C + 8 accumulations loses at most 2 u of the running
  sum (tensor-core accumulation may truncate);
* a probability: the exponent's error (that of its logit and of the row's
  log-sum, and three roundings of |t|), ex2 (4 u) and the row's sum, a chain
  of at most 64 + V / 128 + 8 additions and joins;
* P = u_n (p - [v = y]) is rounded to the planes of its type before the
  gradients' products: half a step of bf16 (2^-8) for bf16, 2^-16 for fp16
  (two planes), u for fp32 (three), and with reduction "none" once more by
  the upstream factor;
* a gradient is a sum of K such products: at most K accumulations that lose
  2 u each (a matrix instruction adds 16 products at a time, in up to six
  plane products), three roundings for scale and join, and half a step of its
  type (and at most one subnormal step).
"""

import ctypes
import threading

import pytest
import torch

import gswarp_b200 as gs
from gswarp_b200 import _lib
from gswarp_b200 import _pipeline as pl

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
P_ROUNDING = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -16}


def reference(x, w, y, b=None, ignore=-100, reduction="mean", upstream=None):
    """Loss and gradients of rows x (N, C) in 64 bits, and the bounds of their errors."""
    dtype = x.dtype
    X, W, Y = x.detach().double(), w.detach().double(), y.reshape(-1).long()
    N, V, C = X.shape[0], W.shape[0], X.shape[1]
    B = b.detach().double() if b is not None else torch.zeros(V, dtype=torch.float64, device=X.device)
    masked = B == -float("inf")
    W = torch.where(masked[:, None], 0.0, W)
    valid = Y != ignore
    at = torch.where(valid, Y, 0)
    dead = valid & masked[at]                      # +inf loss, no gradient
    live = valid & ~dead
    X = torch.where(valid[:, None], X, 0.0)
    z = X @ W.T + B
    ez = ((C + 8) * 2 * U * (X.abs() @ W.abs().T + B.abs()) + 3 * U * z.abs())
    ez = torch.where(masked, 0.0, ez).amax(1)      # the row's worst logit
    lse = torch.logsumexp(z, 1)
    logp = z - lse[:, None]
    chain = (64 + V / 128 + 8) * U
    rows = torch.where(live, -logp.gather(1, at[:, None])[:, 0], 0.0)
    rows = torch.where(dead, float("inf"), rows)
    e_rows = torch.where(live, 2 * ez + chain + 4 * U + 2 * U * rows, 0.0)
    count = valid.sum().clamp(min=1).double()
    out = {}
    if reduction == "none":
        out["loss"] = rows, e_rows
    else:
        f = 1.0 if reduction == "sum" else 1.0 / count
        out["loss"] = rows.sum() * f, (e_rows.sum() + 2 * U * rows.sum()) * f
    if upstream is not None:
        u = upstream.detach().double().reshape(-1).expand(N) / (count if reduction == "mean" else 1.0)
        u = torch.where(live, u, 0.0)[:, None]
        p = logp.exp()
        Pm = p.clone()
        Pm[torch.arange(N), at] = torch.expm1(logp[torch.arange(N), at])
        Pm = torch.where(live[:, None], Pm, 0.0)
        # relative error of p, then the rounding of P itself (fp32 subtraction: U)
        eP = torch.where(live[:, None], p * (torch.expm1(2 * ez[:, None]) + chain + 8 * U), 0.0)
        # ex2 flushes below 2^-126
        eP = eP + torch.where(live[:, None], 2.0 ** -126, 0.0)
        eP = eP + (P_ROUNDING[dtype] + 2 * U) * 1.01 * (Pm.abs() + eP)
        half = torch.finfo(dtype).eps / 2 * 1.01
        tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
        ua = u.abs()

        def bound(err, mag, value, K, h, t):
            return err + (2 * K + 16) * U * (mag + err) + 4 * U * value.abs() + h * (value.abs() + err) + t

        for name, val, err, mag, K, h, t in (
                ("features", (u * Pm) @ W, (ua * eP) @ W.abs(), (ua * Pm.abs()) @ W.abs(), V, half, tiny),
                ("weight", (u * Pm).T @ X, (ua * eP).T @ X.abs(), (ua * Pm.abs()).T @ X.abs(), N, half, tiny),
                ("bias", (u * Pm).sum(0), (ua * eP).sum(0), (ua * Pm.abs()).sum(0), N, 0.0, 2.0 ** -149)):
            out["grad_" + name] = val, bound(err, mag, val, K, h, t)
    return out


def _inputs(N, C, V, dtype, bias=True, ignore=0.1, seed=0, spread=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = (torch.randn(V, C, generator=g, device="cuda") / C ** 0.5).to(dtype)
    y = torch.randint(0, V, (N,), generator=g, device="cuda")
    x = (spread * w[y].float() + torch.randn(N, C, generator=g, device="cuda")).to(dtype)
    if ignore:
        y[torch.rand(N, generator=g, device="cuda") < ignore] = -100
    b = torch.randn(V, generator=g, device="cuda") if bias else None
    return x, w, y, b


def _run(x, w, y, b=None, reduction="mean", upstream=None, **kw):
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b) if t is not None]
    loss = gs.class_cross_entropy(leaves[0], leaves[1], y, leaves[2] if b is not None else None,
                                  reduction=reduction, **kw)
    out = {"loss": loss.detach()}
    if upstream is not None:
        grads = torch.autograd.grad(loss, leaves, upstream)
        out.update(zip(("grad_features", "grad_weight", "grad_bias"), grads))
    return out


def _compare(got, want):
    for k, v in got.items():
        ref, tol = want[k]
        v = v.double().reshape(ref.shape)
        same_inf = torch.isinf(ref) & (v == ref)
        bad = ~(((v - ref).abs() <= tol) | same_inf)
        assert not bad.any(), (k, int(bad.sum()), float(((v - ref).abs() / tol)[bad].max()))


def _upstream(reduction, N, seed=7):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.rand(N if reduction == "none" else (), generator=g, device="cuda") + 0.5


SIZES = [(1, 1, 1), (1, 16, 2), (2, 3, 127), (127, 16, 128), (128, 17, 129), (129, 15, 255), (130, 32, 256),
         (257, 33, 257), (300, 64, 384), (255, 65, 385), (1000, 16, 300), (5, 128, 5000), (4099, 3, 7), (700, 100, 513)]


@pytest.mark.parametrize("N, C, V", SIZES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_against_the_definition(cuda, N, C, V, dtype, reduction):
    x, w, y, b = _inputs(N, C, V, dtype, bias=(N + V) % 2 == 0, seed=N + C + V)
    if N == 1:
        y.fill_(V - 1)
    up = _upstream(reduction, N)
    _compare(_run(x, w, y, b, reduction, up), reference(x, w, y, b, -100, reduction, up))


@pytest.mark.parametrize("N, C, V", [(150, 129, 300), (257, 200, 129), (130, 256, 515), (70, 255, 1000)])
@pytest.mark.parametrize("dtype", TYPES[1:])
def test_wide_features_in_16_bits(cuda, N, C, V, dtype):
    x, w, y, b = _inputs(N, C, V, dtype, seed=C)
    up = _upstream("mean", N)
    _compare(_run(x, w, y, b, "mean", up), reference(x, w, y, b, -100, "mean", up))


@pytest.mark.parametrize("N, C, V, dtype", [(40_000, 16, 256, torch.float32), (33_333, 32, 100, torch.bfloat16),
                                            (20_011, 64, 129, torch.float16), (3, 16, 60_001, torch.float32),
                                            (700, 48, 20_000, torch.bfloat16)])
def test_many_rows_and_many_classes(cuda, N, C, V, dtype):
    x, w, y, b = _inputs(N, C, V, dtype, seed=V)
    up = _upstream("mean", N)
    _compare(_run(x, w, y, b, "mean", up), reference(x, w, y, b, -100, "mean", up))


@pytest.mark.parametrize("shape", [(16, 9, 31), (2, 5, 17, 40), (3, 33, 1, 130), (1, 1, 20, 20), (4, 8, 7, 1)])
@pytest.mark.parametrize("dtype", TYPES)
def test_maps_and_their_strides(cuda, shape, dtype):
    B, (C, H, W) = (1, shape) if len(shape) == 3 else (shape[0], shape[1:])
    V = 140
    rows, w, y, b = _inputs(B * H * W, C, V, dtype, seed=C)
    up = _upstream("mean", 1)
    want = reference(rows, w, y, b, -100, "mean", up)
    first = rows.reshape(B, H, W, C).permute(0, 3, 1, 2)
    first = first[0] if len(shape) == 3 else first
    labels = y.reshape(first.shape[:-3] + (H, W))
    padded = torch.zeros(*first.shape[:-1], W + 3, dtype=dtype, device=cuda)
    padded[..., :W] = first
    twice = torch.zeros(*first.shape[:-1], 2 * W, dtype=dtype, device=cuda)
    twice[..., ::2] = first
    for x in (first.contiguous(), first, padded[..., :W], twice[..., ::2]):
        assert torch.equal(x, first)
        got = _run(x, w, labels, b, "mean", up)
        assert got["grad_features"].shape == first.shape
        g = got["grad_features"]
        g = (g[None] if g.ndim == 3 else g).permute(0, 2, 3, 1)
        _compare({**got, "grad_features": g.reshape(-1, C)}, want)


def test_rows_strides_types_of_labels_and_weights(cuda):
    x, w, y, b = _inputs(300, 20, 77, torch.bfloat16, seed=3)
    up = _upstream("sum", 300)
    want = reference(x, w, y, b, -100, "sum", up)
    wide = torch.zeros(300, 53, dtype=x.dtype, device=cuda)
    wide[:, 5:25] = x
    wt = w.t().contiguous().t()
    y2 = torch.stack([y, y], 1)[:, 0]
    b2 = torch.stack([b, b], 1)[:, 1]
    for x2 in (x, wide[:, 5:25], x.t().contiguous().t()):
        for y3 in (y, y.int(), y2):
            _compare(_run(x2, wt, y3, b2, "sum", up), want)


def test_only_the_wanted_gradients(cuda):
    x, w, y, b = _inputs(200, 16, 150, torch.float32, seed=4)
    up = _upstream("mean", 200)
    full = _run(x, w, y, b, "mean", up)
    for k in ("features", "weight", "bias"):
        t = {"features": x, "weight": w, "bias": b}
        t[k] = t[k].clone().requires_grad_(True)
        g, = torch.autograd.grad(gs.class_cross_entropy(t["features"], t["weight"], y, t["bias"]), t[k], up)
        assert torch.equal(g, full["grad_" + k])
    loss = gs.class_cross_entropy(x.requires_grad_(True), w, y, b, train=False)
    assert torch.equal(loss.detach(), full["loss"])


@pytest.mark.parametrize("N, C, V", SIZES + [(300, 256, 700), (40_000, 16, 513)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_a_forward_alone(cuda, N, C, V, dtype, reduction):
    if C > 128 and dtype == torch.float32:
        pytest.skip("fp32 features have at most 128 channels")
    x, w, y, b = _inputs(N, C, V, dtype, bias=(N + V) % 2 == 0, seed=N + C + V)
    x, w = x.requires_grad_(True), w.requires_grad_(True)
    loss = gs.class_cross_entropy(x, w, y, b, reduction=reduction, train=False)
    assert not loss.requires_grad
    _compare({"loss": loss}, reference(x, w, y, b, -100, reduction))


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_no_row_left(cuda, reduction):
    x, w, y, b = _inputs(300, 16, 150, torch.float32)
    y.fill_(-100)
    x[5] = float("nan")
    got = _run(x, w, y, b, reduction, _upstream(reduction, 300))
    for v in got.values():
        assert (v == 0).all()


def test_no_rows_at_all(cuda):
    _, w, _, b = _inputs(1, 16, 150, torch.float32)
    for shape, lab in (((0, 16), (0,)), ((2, 16, 0, 5), (2, 0, 5))):
        for reduction in ("mean", "sum", "none"):
            x = torch.empty(shape, device=cuda)
            y = torch.empty(lab, dtype=torch.int64, device=cuda)
            up = torch.ones(lab if reduction == "none" else (), device=cuda)
            got = _run(x, w, y, b, reduction, up)
            assert got["grad_features"].shape == shape and (got["grad_weight"] == 0).all()
            assert (got["grad_bias"] == 0).all() and (got["loss"] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_what_ignored_rows_hold_does_not_matter(cuda, dtype):
    x, w, y, b = _inputs(400, 20, 150, dtype, ignore=0.3, seed=6)
    up = _upstream("none", 400)
    ref = _run(x, w, y, b, "none", up)
    x2, up2 = x.clone(), up.clone()
    gone = y == -100
    x2[gone] = float("nan")
    x2[torch.nonzero(gone)[0]] = float("inf")
    up2[gone] = float("nan")
    got = _run(x2, w, y, b, "none", up2)
    for k in ref:
        assert torch.equal(got[k], ref[k]), k


@pytest.mark.parametrize("mask", [-float("inf"), torch.finfo(torch.float32).min])
def test_masked_classes(cuda, mask):
    x, w, y, b = _inputs(300, 16, 260, torch.float32, seed=8)
    off = torch.zeros(260, dtype=torch.bool, device=cuda)
    off[::3] = True
    off[128:256] = True
    b = torch.where(off, mask, b)
    y = torch.where((y >= 0) & off[y.clamp(min=0)], 1, y)
    w2 = w.clone()
    if mask == -float("inf"):
        w2[off] = float("nan")          # their rows are not read
    up = _upstream("mean", 300)
    got = _run(x, w2, y, b, "mean", up)
    want = reference(x, w, y, torch.where(off, -float("inf"), b), -100, "mean", up)
    _compare(got, want)
    assert (got["grad_weight"][off] == 0).all() and (got["grad_bias"][off] == 0).all()


def test_a_label_whose_class_is_masked(cuda):
    x, w, y, b = _inputs(200, 16, 140, torch.float32, ignore=0.0, seed=9)
    b[130] = -float("inf")
    y[17] = 130
    up = _upstream("none", 200)
    got = _run(x, w, y, b, "none", up)
    assert got["loss"][17] == float("inf") and (got["grad_features"][17] == 0).all()
    _compare(got, reference(x, w, y, b, -100, "none", up))
    b.fill_(-float("inf"))              # nothing is left of any row
    got = _run(x, w, y, b, "none", up)
    assert (got["loss"] == float("inf")).all()
    assert all((got["grad_" + k] == 0).all() for k in ("features", "weight", "bias"))


def test_every_class_at_the_lowest_value(cuda):
    x, w, y, _ = _inputs(64, 16, 50, torch.float32, ignore=0.0)
    b = torch.full((50,), torch.finfo(torch.float32).min, device=cuda)
    loss = gs.class_cross_entropy(x, w, y, b, reduction="none")
    # the logits all round to one value: log 50, exact to the roundings of a sum of 50 ones and a logarithm
    assert ((loss.double() - torch.log(torch.tensor(50.0, dtype=torch.float64))).abs() <= 64 * U).all()


@pytest.mark.parametrize("dtype, scale", [(torch.float32, 1e4), (torch.bfloat16, 200.0), (torch.float16, 100.0)])
def test_large_logits(cuda, dtype, scale):
    x, w, y, b = _inputs(200, 16, 300, dtype, seed=10)
    x = (x.float() * scale).to(dtype)
    up = _upstream("mean", 200)
    got = _run(x, w, y, b, "mean", up)
    assert all(torch.isfinite(v).all() for v in got.values())
    loss, tol = reference(x, w, y, b, -100, "mean")["loss"]
    assert abs(float(got["loss"]) - float(loss)) <= float(tol)


def test_nan_and_infinite_features_stay_in_their_rows(cuda):
    x, w, y, b = _inputs(300, 16, 150, torch.float32, ignore=0.0, seed=11)
    ref = _run(x, w, y, b, "none", _upstream("none", 300))
    x[3], x[200, 5] = float("nan"), float("inf")
    got = _run(x, w, y, b, "none", _upstream("none", 300))
    keep = torch.ones(300, dtype=torch.bool, device=cuda)
    keep[[3, 200]] = False
    assert torch.equal(got["loss"][keep], ref["loss"][keep])
    assert torch.equal(got["grad_features"][keep], ref["grad_features"][keep])
    assert torch.isnan(got["loss"][3])


@pytest.mark.parametrize("bad", [-1, 150, 2 ** 33, -2 ** 40])
def test_labels_out_of_range_are_reported(cuda, bad):
    pl.raise_device_errors(cuda)
    x, w, y, b = _inputs(300, 16, 150, torch.float32, seed=12)
    up = _upstream("mean", 300)
    y[100] = bad
    got = _run(x, w, y, b, "mean", up)
    with pytest.raises(RuntimeError, match="label"):
        pl.raise_device_errors(cuda)
    y[100] = -100
    ref = _run(x, w, y, b, "mean", up)
    pl.raise_device_errors(cuda)
    assert all(torch.equal(got[k], ref[k]) for k in ref)


def test_another_ignore_index(cuda):
    x, w, y, b = _inputs(300, 16, 150, torch.float32, ignore=0.0, seed=13)
    up = _upstream("mean", 300)
    _compare(_run(x, w, y, b, "mean", up, ignore_index=3), reference(x, w, y, b, 3, "mean", up))


@pytest.mark.parametrize("N, C, V, dtype", [(5000, 16, 300, torch.float32), (300, 64, 9000, torch.bfloat16)])
def test_the_same_bits_on_every_call(cuda, N, C, V, dtype):
    x, w, y, b = _inputs(N, C, V, dtype, seed=14)
    up = _upstream("mean", N)
    a, c = _run(x, w, y, b, "mean", up), _run(x, w, y, b, "mean", up)
    assert all(torch.equal(a[k], c[k]) for k in a)


def test_gradients_against_differences(cuda):
    x, w, y, b = _inputs(60, 8, 40, torch.float32, seed=15, spread=1.0)
    up = torch.ones((), device=cuda)
    got = _run(x, w, y, b, "sum", up)
    f = lambda *t: reference(*t, -100, "sum")["loss"][0]  # noqa: E731
    h = 1e-4
    for k, i in (("features", 0), ("weight", 1), ("bias", 3)):
        args = [x.double(), w.double(), y, b.double()]
        d = torch.randn_like(args[i])
        hi, lo = list(args), list(args)
        hi[i], lo[i] = args[i] + h * d, args[i] - h * d
        want = float((f(*hi) - f(*lo)) / (2 * h))
        # the difference quotient in 64 bits is off by h^2 / 6 of the third derivative (below 60 rows x
        # |d|^3 <= 60 * 20^3); the kernel's gradient by its own bound
        _, tol = reference(x, w, y, b, -100, "sum", up)["grad_" + k]
        slack = float((tol * d.abs()).sum()) + h * h * 60 * 20 ** 3
        assert abs(float((got["grad_" + k].double() * d).sum()) - want) <= slack


def test_live_graphs_streams_and_retained_graphs(cuda):
    a = _inputs(700, 16, 300, torch.float32, seed=16)
    c = _inputs(500, 48, 200, torch.bfloat16, seed=17)
    up = _upstream("mean", 1)
    ref = [_run(*a, "mean", up), _run(*c, "mean", up)]
    torch.cuda.synchronize()
    leaves, losses = [], []
    for x, w, y, b in (a, c):
        ls = [t.detach().requires_grad_(True) for t in (x, w, b)]
        leaves.append(ls)
        losses.append(gs.class_cross_entropy(ls[0], ls[1], y, ls[2]))
    for k in (1, 0):  # both forwards are alive before either backward
        for _ in range(2):
            g = torch.autograd.grad(losses[k], leaves[k], up, retain_graph=True)
            assert all(torch.equal(p, ref[k][n]) for p, n in zip(g, ("grad_features", "grad_weight", "grad_bias")))
    got = [None, None]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for k, t in enumerate((a, c)):
        streams[k].wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(streams[k]):
            got[k] = _run(*t, "mean", up)
    torch.cuda.synchronize()
    for k in (0, 1):
        assert all(torch.equal(got[k][n], ref[k][n]) for n in ref[k])


def test_captured_and_replayed(cuda):
    x, w, y, b = _inputs(900, 16, 300, torch.float32, seed=18)
    up = _upstream("mean", 1)
    _run(x, w, y, b, "mean", up)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _run(x, w, y, b, "mean", up)
        graphs.append((g, out))
    for seed in (19, 20):
        new = _inputs(900, 16, 300, torch.float32, seed=seed)
        for t, n in zip((x, w, y, b), new):
            t.copy_(n)
        want = _run(*new, "mean", up)
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(out[k], want[k]) for k in want)


@pytest.mark.parametrize("rows", [False, True])
def test_offsets_past_32_bits(cuda, rows):
    C, H, W, V = 256, 2900, 2900, 40  # 2.15e9 elements; the last 3 image rows count
    g = torch.Generator(device="cuda").manual_seed(0)
    N, tail = H * W, 3 * W
    x = torch.zeros((N, C) if rows else (C, H, W), dtype=torch.bfloat16, device=cuda)
    last = torch.randn(tail, C, generator=g, device="cuda").bfloat16()
    if rows:
        x[N - tail:] = last
    else:
        x[:, H - 3:] = last.t().reshape(C, 3, W)
    w = (torch.randn(V, C, generator=g, device="cuda") / 16).bfloat16()
    y = torch.full((N,), -100, device=cuda)
    y[N - tail:] = torch.randint(0, V, (tail,), generator=g, device="cuda")
    up = torch.ones((), device=cuda)
    got = _run(x, w, y if rows else y.view(H, W), None, "mean", up)
    gx = got["grad_features"]
    head, end = (gx[:N - tail], gx[N - tail:]) if rows else (gx[:, :H - 3], gx[:, H - 3:].reshape(C, tail).t())
    assert not head.any()
    _compare({**got, "grad_features": end}, reference(last, w, y[N - tail:], None, -100, "mean", up))


def test_a_scene_with_shared_feature_rows_is_trained_through_both(cuda):
    """Codebook rows -> rasterizer -> class loss, and back to the codebook."""
    from gswarp_b200 import workloads as wl

    scene, view = wl.config1_scene(seed=0, n=2000)
    s, v = scene.to(cuda), view.to(cuda)
    settings = gs.GaussianRasterizationSettings(
        image_height=v.height, image_width=v.width, tanfovx=v.tanfovx, tanfovy=v.tanfovy,
        bg=torch.zeros(3, device=cuda), scale_modifier=1.0, viewmatrix=v.viewmatrix, projmatrix=v.projmatrix,
        sh_degree=0, campos=v.campos, prefiltered=False)
    g = torch.Generator(device="cuda").manual_seed(0)
    table = torch.randn(64, 6, generator=g, device="cuda", requires_grad=True)
    codes = torch.randint(0, 64, (2000,), generator=g, device="cuda")
    weight = torch.randn(30, 6, generator=g, device="cuda", requires_grad=True)
    labels = torch.randint(0, 30, (v.height, v.width), generator=g, device="cuda")
    feats = gs.codebook_lookup(table, codes)
    feats.retain_grad()
    maps = [gs.GaussianRasterizer(settings)(s.means, torch.zeros_like(s.means), s.opacities,
                                            colors_precomp=feats[:, k:k + 3].contiguous(), scales=s.scales,
                                            rotations=s.rotations)[0] for k in (0, 3)]
    image = torch.cat(maps)
    image.retain_grad()
    loss = gs.class_cross_entropy(image, weight, labels)
    loss.backward()
    rows = image.detach().permute(1, 2, 0).reshape(-1, 6)
    want = reference(rows, weight, labels, None, -100, "mean", torch.ones((), device=cuda))
    _compare({"loss": loss.detach(), "grad_weight": weight.grad,
              "grad_features": image.grad.permute(1, 2, 0).reshape(-1, 6)}, want)
    # rows of one code: 2000 Gaussians, sums of at most 2000 terms
    ref, mag = torch.zeros(64, 6, dtype=torch.float64, device=cuda), torch.zeros(64, 6, dtype=torch.float64,
                                                                               device=cuda)
    ref.index_add_(0, codes, feats.grad.double())
    mag.index_add_(0, codes, feats.grad.double().abs())
    assert float(mag.max()) > 0
    assert ((table.grad.double() - ref).abs() <= 300 * U * mag + 2.0 ** -149).all()


@pytest.mark.parametrize("dtype", TYPES[:2])
def test_a_label_whose_logit_overflows_keeps_its_gradient(cuda, dtype):
    # z[17, 130] = -2^200 is -inf in fp32; the class takes part, so P[17, 130] is softmax 0 less 1
    x, w, y, b = _inputs(200, 16, 140, dtype, ignore=0.0, seed=19)
    x[:, 0], w[:, 0] = 0.0, 0.0
    x[17, 0], w[130, 0], y[17] = 2.0 ** 100, -2.0 ** 100, 130
    up = _upstream("none", 200)
    got = _run(x, w, y, b, "none", up)
    assert got["loss"][17] == float("inf")
    z = x[17].double() @ w.double().T + b.double()
    p = torch.softmax(z, 0)
    p[130] -= 1.0
    u = up[17].double()
    # a logit of at most 10 in magnitude: (C + 8) * 2 U * 40 for the products' magnitudes and the chain of the row's
    # sum, 2 (64 + 10) U; P's rounding; half a step of the result; 140 products added up
    err = (24 * 2 * U * 40 + 150 * U + P_ROUNDING[dtype] + 2 * 140 * U)
    mag = (p.abs() @ w.double().abs()) * u
    tol = 1.01 * (err * mag + torch.finfo(dtype).eps / 2 * ((p @ w.double()) * u).abs())
    assert ((got["grad_features"][17].double() - (p @ w.double()) * u).abs() <= tol).all()
    assert float(got["grad_features"][17].abs().max()) > 0
    # the class's gradient has the row: -u x[17, 0] and nothing else in that column
    want = -u * 2.0 ** 100
    assert abs(float(got["grad_weight"][130, 0].double() - want)) <= 1.01 * (
        P_ROUNDING[dtype] + 2 * U + torch.finfo(dtype).eps / 2) * abs(float(want)) * 2


@pytest.mark.parametrize("dtype", TYPES)
def test_two_host_threads_with_different_channels(cuda, dtype):
    """Calls of the C ABI side by side: one kernel instantiation, two plans of shared memory."""
    up = _upstream("mean", 1)
    calls, want, held = [], [], []
    for C, seed in ((16, 20), (64, 21)):
        x, w, y, b = _inputs(300, C, 200, dtype, seed=seed)
        want.append(_run(x, w, y, b, "mean", up))
        a = _lib.ClassLossArgs(1, 300, 200, C, _lib.DTYPES[dtype], 2, 1, 1, 0, 1, C, -100, x.data_ptr(), w.data_ptr(),
                               b.data_ptr(), y.data_ptr())
        sizes = (ctypes.c_size_t * 3)()
        _lib.call("gsb_class_loss_sizes", a, sizes)
        kept, ws = (torch.empty(n, dtype=torch.uint8, device=cuda) for n in (sizes[0], max(sizes[1], sizes[2])))
        out = {"loss": torch.empty(1, device=cuda), "grad_features": torch.empty_like(x),
               "grad_weight": torch.empty_like(w), "grad_bias": torch.empty_like(b)}
        a.kept, a.workspace, a.workspace_bytes = kept.data_ptr(), ws.data_ptr(), ws.numel()
        a.loss, a.upstream, a.error_word = out["loss"].data_ptr(), up.data_ptr(), pl.sticky_error_word(cuda).data_ptr()
        a.grad_features, a.grad_weight = out["grad_features"].data_ptr(), out["grad_weight"].data_ptr()
        a.grad_bias = out["grad_bias"].data_ptr()
        calls.append((a, out))
        held.append((x, w, y, b, kept, ws))
    torch.cuda.synchronize()
    failed, start = [], threading.Barrier(2)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    L = _lib.load()

    def work(k):
        a, stream = calls[k][0], streams[k].cuda_stream
        torch.cuda.set_device(cuda)
        start.wait(30)
        for _ in range(1000):
            if L.gsb_class_loss_fwd(a, stream) or L.gsb_class_loss_bwd(a, stream):
                failed.append((k, L.gsb_last_error()))
                return

    threads = [threading.Thread(target=work, args=(k,)) for k in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed
    for (_, out), ref in zip(calls, want):
        assert all(torch.equal(out[n].view_as(ref[n]), ref[n]) for n in ref)


@pytest.mark.parametrize("dtype", TYPES)
def test_no_gradient_wanted_is_a_forward_alone(cuda, dtype, monkeypatch):
    x, w, y, b = _inputs(300, 20, 150, dtype, seed=22)
    want = reference(x, w, y, b, -100, "mean")
    trained, call_on = [], _lib.call_on

    def spy(dev, name, a):
        trained.append(a.train)
        call_on(dev, name, a)

    monkeypatch.setattr(_lib, "call_on", spy)
    losses = [gs.class_cross_entropy(x, w, y, b)]
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    with torch.no_grad():
        losses.append(gs.class_cross_entropy(leaves[0], leaves[1], y, leaves[2]))
    for k in range(3):  # one leaf is enough
        a, c, d = (leaves[i] if i == k else t for i, t in enumerate((x, w, b)))
        losses.append(gs.class_cross_entropy(a, c, y, d))
    assert trained == [0, 0, 1, 1, 1] and [t.requires_grad for t in losses] == [False, False, True, True, True]
    for loss in losses:
        _compare({"loss": loss.detach()}, want)


def test_a_program_of_the_loss_alone_learns_of_a_bad_label(cuda):
    gs.raise_device_errors()
    x, w, y, b = _inputs(300, 16, 150, torch.float32, seed=23)
    y[7] = 150
    gs.class_cross_entropy(x, w, y, b)
    for device in (None, cuda, str(cuda), torch.cuda.current_device()):
        y[7] = 150
        gs.class_cross_entropy(x, w, y, b)
        with pytest.raises(RuntimeError, match="class label out of range"):
            gs.raise_device_errors(device)
        gs.raise_device_errors(device)


def _exact(x, w, y):
    """dX and dW of the summed loss in 64 bits, by pieces of rows."""
    X, W = x.double(), w.double()
    dX, dW = torch.empty_like(X), torch.zeros_like(W)
    piece = max(1, 100_000_000 // W.shape[0])
    for lo in range(0, X.shape[0], piece):
        rows = X[lo:lo + piece]
        p = torch.log_softmax(rows @ W.T, 1)
        at = torch.arange(len(rows), device=x.device), y[lo:lo + piece]
        label = torch.expm1(p[at])
        p.exp_()
        p[at] = label
        dX[lo:lo + piece] = p @ W
        dW += p.T @ rows
    return dX, dW


def _off(got, want):
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.parametrize("N, C, V, dtype, most", [
    (100_000, 5, 15, torch.bfloat16, 1.1), (100_000, 2, 149, torch.bfloat16, 1.1),     # two planes of P
    (50_000, 32, 1000, torch.bfloat16, 1.8),                                           # one
    (100_000, 16, 300, torch.float16, 1.1), (30_000, 200, 700, torch.float16, 1.1),
])
def test_gradients_are_off_by_little_more_than_their_own_rounding(cuda, N, C, V, dtype, most):
    """Norms of the error over norms of the gradients' rounding to their type.  What comes before that rounding is
    2^-16 of a product and less where P has two planes, which is 2^-8 of the rounding of bf16 and 2^-5 of that of fp16.
    One plane of bf16 rounds each product as the result is rounded: sqrt(2) in all where products do not cancel, and
    the label's term takes away up to as much again of the result."""
    x, w, y, _ = _inputs(N, C, V, dtype, bias=False, ignore=0.0, seed=24, spread=1.0)
    got = _run(x, w, y, None, "sum", torch.ones((), device=cuda))
    for name, want in zip(("grad_features", "grad_weight"), _exact(x, w, y)):
        assert _off(got[name], want) <= most * _off(want.to(dtype), want), name


def test_the_error_of_fp32_gradients(cuda):
    """Norm of the error over the norm of the gradients, 100,000 rows, logits of magnitude 1 and |t| below 16 in base
    2.  Rounding the exponent twice and the row's log-sum once, 2^-20 / sqrt(12) ln 2 each: 3.3e-7 together; ex2 2^-23;
    16 additions that truncate before a sum is taken out, half an ulp of 2^-23 on average: 16 * 2^-24; then sums that
    are rounded, the logits' products and the planes, below 2^-24 each."""
    x, w, y, _ = _inputs(100_000, 16, 256, torch.float32, bias=False, ignore=0.0, seed=25, spread=0.0)
    w *= 0.3
    got = _run(x, w, y, None, "sum", torch.ones((), device=cuda))
    for name, want in zip(("grad_features", "grad_weight"), _exact(x, w, y)):
        assert _off(got[name], want) <= 16 * U + 3.3e-7 + 2 * U + 3 * U, name


@pytest.mark.parametrize("dtype, chain", [(torch.float32, 16), (torch.float16, 256), (torch.bfloat16, 512)])
@pytest.mark.parametrize("which", ["grad_weight", "grad_features"])
def test_long_sums_do_not_drift(cuda, dtype, chain, which):
    """Sums of 50,000 to 300,000 products of one sign: a chain of additions that truncate loses half an ulp of 2^-23 of
    its running sum each, always the same way, and is cut after `chain` of them.  The mean relative error of all
    elements, from which their own rounding (half a step, uniform) goes as 1 / sqrt(n): five standard deviations of
    it, the chain, and 3e-6 for the probabilities (ex2 2^-22, the truncated products of logits below 2 in magnitude)."""
    g = torch.Generator(device="cuda").manual_seed(26)
    if which == "grad_weight":
        N, C, V = 300_000, 64, 512
    else:
        N, C, V = 148 * 128, 16, 200_000 if dtype == torch.bfloat16 else 50_000   # one unit per SM, over all classes
    y = torch.zeros(N, dtype=torch.int64, device=cuda)
    x, w = torch.randn(N, C, generator=g, device=cuda), torch.randn(V, C, generator=g, device=cuda)
    if which == "grad_weight":
        x, w = 0.1 + x.abs(), 0.05 * w
    else:
        x, w = 0.1 * x, 0.1 + w.abs()
        w[0] = 0.0          # the label's class adds nothing
    x, w = x.to(dtype), w.to(dtype)
    got = _run(x, w, y, None, "sum", torch.ones((), device=cuda))[which].double()
    want = _exact(x, w, y)[which == "grad_weight"]
    if which == "grad_weight":
        got, want = got[1:], want[1:]                       # the other classes' rows are positive
    assert (want > 0).all()
    drift = abs(float(((got - want) / want).mean()))
    assert drift <= chain * U + 5 * torch.finfo(dtype).eps / 2 / 3 ** 0.5 / want.numel() ** 0.5 + 3e-6


@pytest.mark.parametrize("dtype, scale", [(torch.float32, 1e4), (torch.float32, 100.0), (torch.bfloat16, 200.0),
                                          (torch.bfloat16, 20.0), (torch.float16, 100.0), (torch.float16, 10.0)])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_gradients_at_large_logits(cuda, dtype, scale, reduction):
    x, w, y, b = _inputs(200, 16, 300, dtype, seed=10)
    x = (x.float() * scale).to(dtype)
    up = _upstream(reduction, 200)
    _compare(_run(x, w, y, b, reduction, up), reference(x, w, y, b, -100, reduction, up))


@pytest.mark.parametrize("N, C, V", [(20_000, 16, 2), (20_000, 16, 8), (64, 1, 3)])
def test_the_planes_of_fp32_probabilities(cuda, N, C, V):
    """Norm of dX's error over its own, few classes and logits below 1 in magnitude, so that |t| < 4 in base 2: three
    roundings of 2^-23 ln 2 in the exponent, ex2 2^-22, four truncations of an ulp of 2^-23 in the logits' and the
    gradients' last products, three roundings.  1.1e-6 in all; without its third plane P alone would be off by
    2^-18 / sqrt(3) = 2.2e-6."""
    x, w, y, _ = _inputs(N, C, V, torch.float32, bias=False, ignore=0.0, seed=27, spread=0.0)
    w *= 0.3
    got = _run(x, w, y, None, "sum", torch.ones((), device=cuda))["grad_features"]
    assert _off(got, _exact(x, w, y)[0]) <= 3 * 2 * U * 0.6931 + 4 * U + 4 * 2 * U + 3 * U
