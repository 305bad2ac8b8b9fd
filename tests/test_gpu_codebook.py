"""codebook_lookup against its definition in 64 bits.

Tolerances count roundings.  A row element is scale * gain (one rounding of
2^-24), times the table entry (one more), rounded to the table's type (half a
step).  A gradient element is a sum of n products s * g: each product carries
at most three roundings of 2^-24, and each summand passes through at most
min(n, DEPTH) additions (chunks of at most 128 rows, then the chunks of a run,
which eight warps share: at most 340 of each here, the longest run being a
third of 1.06M rows in chunks of 128), each one rounding of the running sum,
which the sum of magnitudes bounds.  A gain's gradient is a dot product of D
terms times scale.
"""

import pytest
import torch

import gswarp_b200 as gs
from gswarp_b200 import _pipeline as pl
from gswarp_b200 import codebook

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DEPTH = 128 + 340
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _tiny(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps  # one subnormal step


def _inputs(P, K, D, dtype, index=torch.int64, gain=True, seed=0, unassigned=0.1, skew=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    table = torch.randn(K, D, generator=g, device="cuda").to(dtype)
    codes = (K * torch.rand(P, generator=g, device="cuda").double() ** skew).long().clamp(max=max(K - 1, 0))
    if unassigned:
        codes = torch.where(torch.rand(P, generator=g, device="cuda") < unassigned, -1, codes)
    s = torch.exp(0.5 * torch.randn(P, generator=g, device="cuda")) if gain else 0.75
    up = torch.randn(P, D, generator=g, device="cuda").to(dtype)
    return table, codes.to(index), s, up


def _check(table, codes, scale, up, rows, grad_table, grad_gain):
    dtype = table.dtype
    T, c, g = table.detach().double(), codes.long().reshape(-1), up.double().reshape(codes.numel(), -1)
    T2 = T.reshape(T.shape[0], -1)
    gain = isinstance(scale, torch.Tensor)
    s = scale.detach().double().reshape(-1) if gain else torch.full((c.numel(),), scale, device=c.device,
                                                                     dtype=torch.float64)
    used = c >= 0
    ref = torch.zeros_like(g)
    ref[used] = T2[c[used]] * s[used, None]
    err = (rows.double().reshape(g.shape) - ref).abs()
    assert (err <= (2 * U + _half_step(dtype)) * 1.01 * ref.abs() + _tiny(dtype)).all()
    assert (rows.reshape(g.shape)[~used] == 0).all()
    if grad_table is not None:
        want, mag = torch.zeros_like(T2), torch.zeros_like(T2)
        want.index_add_(0, c[used], g[used] * s[used, None])
        mag.index_add_(0, c[used], (g[used] * s[used, None]).abs())
        n = torch.bincount(c[used], minlength=T2.shape[0]).clamp(max=DEPTH)[:, None].double()
        bound = (n + 3) * U * 1.01 * mag + _half_step(dtype) * 1.01 * want.abs() + _tiny(dtype)
        assert ((grad_table.double().reshape(T2.shape) - want).abs() <= bound).all()
    if grad_gain is not None:
        want, mag = torch.zeros_like(s), torch.zeros_like(s)
        want[used] = (g[used] * T2[c[used]]).sum(1)
        mag[used] = (g[used] * T2[c[used]]).abs().sum(1)
        assert ((grad_gain.double().reshape(-1) - want).abs() <= (g.shape[1] + 2) * U * 1.01 * mag).all()


def _run(table, codes, scale, up):
    t = table.clone().requires_grad_(True)
    leaves = [t]
    if isinstance(scale, torch.Tensor):
        scale = scale.clone().requires_grad_(True)
        leaves.append(scale)
    out = gs.codebook_lookup(t, codes, scale)
    grads = torch.autograd.grad(out, leaves, up)
    return out.detach(), grads[0], grads[1] if len(grads) > 1 else None


@pytest.mark.parametrize("P, K, D", [
    (1, 1, 1), (1, 7, 3), (2, 1, 48), (31, 2, 3), (32, 5, 4), (33, 5, 45), (64, 64, 16), (65, 3, 8), (127, 255, 12),
    (128, 256, 20), (1000, 257, 45), (1025, 1, 48), (4097, 65_537, 3), (10_000, 256, 3), (3841, 700, 77),
    (300, 9, 128), (300, 9, 129), (77, 5, 513), (50, 4, 2001),
    (300, 40_000, 45), (4096, 5000, 8), (3000, 100_000, 140), (1, 9_000_000, 1), (40_000, 900, 12),
])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("gain", [False, True])
def test_against_the_definition(cuda, P, K, D, dtype, gain):
    args = _inputs(P, K, D, dtype, torch.int32 if P % 2 else torch.int64, gain, seed=P + D)
    _check(*args, *_run(*args))


@pytest.mark.parametrize("codes", ["one", "alternating", "none", "each", "ends"])
@pytest.mark.parametrize("D", [3, 48])
def test_distributions_of_codes(cuda, codes, D):
    P, K = 20_011, 4100
    table, c, s, up = _inputs(P, K, D, torch.float32, gain=True)
    i = torch.arange(P, device="cuda")
    c = {"one": torch.full_like(i, 4099), "alternating": i % 2, "none": torch.full_like(i, -1), "each": i % K,
         "ends": torch.where(i < 17, 0, K - 1)}[codes]
    args = (table, c, s, up)
    rows, gt, gg = _run(*args)
    _check(*args, rows, gt, gg)
    if codes == "none":
        assert (gt == 0).all() and (gg == 0).all() and (rows == 0).all()


def test_the_long_chunks_of_many_rows(cuda):
    args = _inputs((1 << 20) + 12_345, 1000, 3, torch.float32, torch.int32, True, seed=9, skew=6.0)
    _check(*args, *_run(*args))


def test_gradients_have_the_same_bits_on_every_call(cuda):
    args = _inputs(200_003, 50, 45, torch.float32, gain=True, seed=3)
    a, b = _run(*args), _run(*args)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_gradient_against_differences(cuda):
    # exact in fp32 up to rounding: the lookup is linear in the table and in the gains
    table, codes, s, up = _inputs(257, 19, 6, torch.float32, seed=5)
    _, gt, gg = _run(table, codes, s, up)
    f = lambda t, g: (gs.codebook_lookup(t, codes, g).double() * up.double()).sum()  # noqa: E731
    dt, dg = torch.randn_like(table), torch.randn_like(s)
    h = 2.0 ** -4
    for got, hi, lo in ((gt.double() @ dt.double().T, f(table + h * dt, s), f(table - h * dt, s)),
                        (None, f(table, s + h * dg), f(table, s - h * dg))):
        want = float((hi - lo) / (2 * h))
        value = float(torch.trace(got)) if got is not None else float((gg.double() * dg.double()).sum())
        # 2 x 1542 rounded products of magnitude |s t up| <= 300 each, divided by 2h
        assert abs(value - want) <= 2 * 1542 * 4 * U * 300 / (2 * h)


def test_shapes_strides_and_views(cuda):
    g = torch.Generator(device="cuda").manual_seed(1)
    big = torch.randn(40, 16, 6, generator=g, device="cuda")
    table = big[::2, :, ::2]                      # (20, 16, 3), not contiguous
    codes = torch.randint(-1, 20, (7, 33), generator=g, device="cuda").t()   # (33, 7), transposed
    gain = torch.rand(7, 33, generator=g, device="cuda").t()
    t = table.clone().requires_grad_(True)
    out = gs.codebook_lookup(table, codes, gain)
    assert out.shape == (33, 7, 16, 3)
    ref = table[codes.clamp(min=0)] * (gain * (codes >= 0))[..., None, None]
    assert torch.equal(out, ref)
    # a broadcast (stride 0) upstream gradient
    gt, = torch.autograd.grad(gs.codebook_lookup(t, codes, gain).sum(), t)
    _check(table, codes, gain, torch.ones(33 * 7, 48, device="cuda"), out, gt, None)
    # an odd element offset breaks 16-byte alignment
    flat = torch.randn(1 + 20 * 48, generator=g, device="cuda").half()
    odd = flat[1:].view(20, 48)
    assert odd.data_ptr() % 16 != 0
    args = (odd, codes.reshape(-1), gain.reshape(-1), torch.randn(231, 48, generator=g, device="cuda").half())
    _check(*args, *_run(*args))


def test_empty_calls(cuda):
    table = torch.randn(5, 3, device="cuda", requires_grad=True)
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    out = gs.codebook_lookup(table, none)
    assert out.shape == (0, 3)
    gt, = torch.autograd.grad(out.sum(), table)
    assert (gt == 0).all()
    empty = torch.empty(0, 3, device="cuda", requires_grad=True)
    out = gs.codebook_lookup(empty, torch.full((4,), -1, device="cuda"))
    assert (out == 0).all() and out.shape == (4, 3)
    gt, = torch.autograd.grad(out.sum(), empty)
    assert gt.shape == (0, 3)


def test_special_values_stay_in_their_rows(cuda):
    table, codes, s, up = _inputs(500, 11, 3, torch.float32, unassigned=0.3, seed=8)
    up[codes == -1] = float("nan")        # rows without a code are not read
    table[4] = float("inf")
    up[codes == 7] = float("nan")
    rows, gt, gg = _run(table, codes, s, up)
    keep = (codes != 4) & (codes >= 0)
    assert torch.isfinite(rows[keep]).all() and (rows[codes == -1] == 0).all()
    assert torch.isinf(rows[codes == 4]).all()
    ok = torch.ones(11, dtype=torch.bool, device="cuda")
    ok[7] = False
    assert torch.isfinite(gt[ok]).all() and torch.isnan(gt[7]).all()
    assert (gg[codes == -1] == 0).all() and torch.isfinite(gg[(codes >= 0) & (codes != 7) & (codes != 4)]).all()


@pytest.mark.parametrize("bad", [-2, 11, 2 ** 31, -2 ** 40])
def test_codes_out_of_range_are_reported(cuda, bad):
    pl.raise_device_errors(cuda)
    table, codes, s, up = _inputs(300, 11, 5, torch.float32, unassigned=0.0, seed=2)
    codes[123] = bad
    rows, gt, gg = _run(table, codes, s, up)
    with pytest.raises(RuntimeError, match="code"):
        pl.raise_device_errors(cuda)
    pl.raise_device_errors(cuda)
    clean = codes.clone()
    clean[123] = -1
    ref = _run(table, clean, s, up)
    pl.raise_device_errors(cuda)
    assert all(torch.equal(a, b) for a, b in zip((rows, gt, gg), ref))


def test_another_stream_and_live_graphs(cuda):
    a1, a2 = _inputs(5000, 60, 45, torch.float32, seed=1), _inputs(7000, 33, 12, torch.bfloat16, seed=2)
    ref1, ref2 = _run(*a1), _run(*a2)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None, None]
    for k, (st, a) in enumerate(zip(streams, (a1, a2))):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            got[k] = _run(*a)
    torch.cuda.synchronize()
    for ref, g in zip((ref1, ref2), got):
        assert all(torch.equal(x, y) for x, y in zip(ref, g))


def test_captured_and_replayed(cuda):
    table, codes, s, up = _inputs(3000, 40, 48, torch.float32, seed=4)
    pl.sticky_error_word(cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        codebook.lookup_backward(table.shape, table.dtype, table, codes, 1.0, s, up, want_gain=True)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):  # two graphs, each with its own workspace
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = (codebook.lookup_forward(table, codes, 1.0, s),
                   *codebook.lookup_backward(table.shape, table.dtype, table, codes, 1.0, s, up, want_gain=True))
        graphs.append((g, out))
    for seed in (11, 12):
        t2, c2, s2, u2 = _inputs(3000, 40, 48, torch.float32, seed=seed)
        table.copy_(t2), codes.copy_(c2), s.copy_(s2), up.copy_(u2)
        want = _run(t2, c2, s2, u2)
        for g, out in graphs:
            g.replay()
        torch.cuda.synchronize()
        for g, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_offsets_past_32_bits(cuda):
    P, D, K = 46_000_003, 48, 5000  # 2.2e9 elements
    g = torch.Generator(device="cuda").manual_seed(0)
    table = torch.randn(K, D, generator=g, device="cuda").bfloat16()
    codes = torch.randint(0, K, (P,), generator=g, device="cuda", dtype=torch.int32)
    out = codebook.lookup_forward(table, codes, 2.0)
    for lo in (0, 44_739_242 - 5, P - 1000):  # the element 2^31 is in row 44,739,242
        n = min(1000, P - lo)
        assert torch.equal(out[lo:lo + n], table[codes[lo:lo + n].long()] * 2)
    # a gradient that is zero but in the last rows
    out.zero_()
    out[P - 1000:] = torch.randn(1000, D, generator=g, device="cuda").bfloat16()
    gt, _ = codebook.lookup_backward(table.shape, table.dtype, None, codes, 2.0, None, out)
    _check(table, codes[P - 1000:], 2.0, out[P - 1000:],
           codebook.lookup_forward(table, codes[P - 1000:].contiguous(), 2.0), gt, None)


def test_the_first_call_on_a_device_is_not_captured(cuda, monkeypatch):
    monkeypatch.setattr(pl, "_STICKY", {})
    table, codes, s, _ = _inputs(100, 5, 3, torch.float32)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="before capturing"):
        with torch.cuda.graph(graph):
            codebook.lookup_forward(table, codes, 1.0, s)


def test_rows_are_rendered_and_the_codebook_gets_the_scenes_gradient(cuda):
    """As it is used: shared SH rows expanded, rendered and trained through the rasterizer."""
    from gswarp_b200 import workloads as wl

    scene, view = wl.config1_scene(seed=0, n=2000)
    s, v = scene.to(cuda), view.to(cuda)
    settings = gs.GaussianRasterizationSettings(
        image_height=v.height, image_width=v.width, tanfovx=v.tanfovx, tanfovy=v.tanfovy,
        bg=torch.zeros(3, device=cuda), scale_modifier=1.0, viewmatrix=v.viewmatrix, projmatrix=v.projmatrix,
        sh_degree=0, campos=v.campos, prefiltered=False)
    g = torch.Generator(device="cuda").manual_seed(0)
    table = torch.randn(64, 1, 3, generator=g, device="cuda", requires_grad=True)
    codes = torch.randint(0, 64, (2000,), generator=g, device="cuda")
    gain = (1 + torch.rand(2000, generator=g, device="cuda")).requires_grad_(True)
    sh = gs.codebook_lookup(table, codes, gain)
    sh.retain_grad()
    target = torch.rand(1, 3, v.height, v.width, generator=g, device="cuda")
    color, _, _ = gs.GaussianRasterizer(settings)(s.means, torch.zeros_like(s.means), s.opacities, shs=sh,
                                                  scales=s.scales, rotations=s.rotations)
    (1 - gs.fused_ssim(color[None], target)).backward()
    assert float(sh.grad.abs().max()) > 0
    _check(table, codes, gain, sh.grad, sh.detach(), table.grad, gain.grad)


def _shared_scene(dev, n, rows, views):
    from gswarp_b200 import workloads as wl

    sc = wl.config2_scene(seed=5, n=n)
    cams = wl.ring_views(views, seed=5, width=320, height=192)
    g = torch.Generator().manual_seed(3)
    table = (0.3 * torch.randn(rows, 16, 3, generator=g)).to(dev)
    codes = torch.randint(-1, rows, (n,), generator=g).to(dev)
    params = [t.to(dev).contiguous() for t in (sc.means, sc.scales, sc.rotations, sc.opacities)]
    settings = [gs.GaussianRasterizationSettings(
        image_height=v.height, image_width=v.width, tanfovx=v.tanfovx, tanfovy=v.tanfovy,
        bg=torch.zeros(3, device=dev), scale_modifier=1.0, viewmatrix=v.viewmatrix.to(dev),
        projmatrix=v.projmatrix.to(dev), sh_degree=3, campos=v.campos.to(dev), prefiltered=False) for v in cams]
    targets = [wl.target_image(100 + i, 192, 320).to(dev) for i in range(views)]
    return params, table, codes, settings, targets


@pytest.mark.parametrize("views, batch_sh", [(1, None), (3, True), (3, False)])
@pytest.mark.parametrize("n", [20_000, 20_003])
def test_fused_step_trains_shared_sh_rows(cuda, views, batch_sh, n):
    from gswarp_b200.training import FusedViewStep

    params, table, codes, settings, targets = _shared_scene(cuda, n, 700, views)
    step = FusedViewStep(params + [table], settings, batch_sh=batch_sh, sh_codes=codes)
    rows = torch.where((codes >= 0)[:, None, None], table[codes.clamp(min=0)], 0.0).contiguous()
    dense = FusedViewStep([p.clone() for p in params] + [rows], settings, batch_sh=batch_sh)
    for _ in range(2):  # a second step starts from zero again
        losses, want = step.step(targets), dense.step(targets)
        # the same rows give the same images
        assert torch.equal(losses, want)
        # the codebook's gradient is the sum of this step's row gradients
        _check(table, codes, 1.0, step._grad_sh_rows, rows, step.grads.views[4], None)
        assert table.grad.data_ptr() == step.grads.views[4].data_ptr()
        # the render backward adds with atomics: blocks of the two runs agree by norm, as between any two runs
        for a, b in zip(step.grads.views[:4], dense.grads.views[:4]):
            assert float((a - b).norm()) <= 1e-4 * float(b.norm()) + 1e-7
        assert float((step._grad_sh_rows - dense.grads.views[4]).norm()) <= 1e-4 * float(dense.grads.views[4].norm())


def test_fused_step_refuses_bad_codes(cuda):
    from gswarp_b200.training import FusedViewStep

    params, table, codes, settings, targets = _shared_scene(cuda, 3000, 50, 2)
    for bad in (codes[:-1], codes.float(), codes.cpu()):
        with pytest.raises(ValueError, match="sh_codes"):
            FusedViewStep(params + [table], settings, sh_codes=bad)
    with pytest.raises(ValueError, match="codebook"):
        FusedViewStep(params + [table[..., :2]], settings, sh_codes=codes)
    with pytest.raises(ValueError, match="fp32 \\(P, K, 3\\)"):
        FusedViewStep(params + [table], settings)
    step = FusedViewStep(params + [table], settings, sh_codes=codes)
    step.deferred_views = 1
    with pytest.raises(ValueError, match="range-ordered"):
        step.step(targets)
    step.deferred_views = 0
    step.step(targets)
    step.sh_codes[5] = 50
    with pytest.raises(RuntimeError, match="code"):
        step.step(targets)
    step.sh_codes[5] = 3
    step.step(targets)


@pytest.mark.parametrize("D", [3, 45, 48])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("P", [300, 20_011])
def test_rows_without_a_code_are_zero_whatever_their_gain_holds(cuda, D, dtype, P):
    table, codes, s, up = _inputs(P, 90, D, dtype, unassigned=0.3, seed=D)
    gone = torch.nonzero(codes == -1)[:, 0]
    s[gone[::3]], s[gone[1::3]] = float("nan"), float("inf")
    rows, gt, gg = _run(table, codes, s, up)
    assert (rows[gone] == 0).all() and (gg[gone] == 0).all()
    clean = torch.where(codes == -1, 1.0, s)
    _check(table, codes, clean, up, rows, gt, gg)
    for number in (float("nan"), float("inf")):
        assert (codebook.lookup_forward(table, codes, number)[gone] == 0).all()
    # a code out of range is no code either
    codes[gone[:3]] = 90
    assert (codebook.lookup_forward(table, codes, 1.0, s)[gone] == 0).all()
    with pytest.raises(RuntimeError, match="code"):
        pl.raise_device_errors(cuda)


@pytest.mark.parametrize("D", [3, 48])
@pytest.mark.parametrize("P", [300, 20_011])
def test_an_infinite_scale_stays_with_the_rows_that_have_a_code(cuda, D, P):
    table, codes, _, _ = _inputs(P, 4100, D, torch.float32, unassigned=0.5, seed=1)
    up = torch.ones(P, D, device="cuda")  # every sum of a code that has rows is +inf
    gt, _ = codebook.lookup_backward(table.shape, table.dtype, None, codes, float("inf"), None, up)
    has = torch.zeros(4100, dtype=torch.bool, device="cuda")
    has[codes[codes >= 0]] = True
    assert (gt[has] == float("inf")).all() and (gt[~has] == 0).all()


def test_a_table_that_backward_does_not_need_may_change(cuda):
    table, codes, s, up = _inputs(500, 11, 6, torch.float32, seed=6)
    want = _run(table, codes, s, up)[1]
    t = table.clone().requires_grad_(True)
    out = gs.codebook_lookup(t, codes, s)       # the gains are fixed: no gradient reads the table
    with torch.no_grad():
        t.add_(1.0)
    got, = torch.autograd.grad(out, t, up)
    assert torch.equal(got, want)
    gain = s.clone().requires_grad_(True)       # the gains' gradient does read it
    out = gs.codebook_lookup(t, codes, gain)
    with torch.no_grad():
        t.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, gain, up)
    out = gs.codebook_lookup(table, codes, gain)   # and not the gains
    want, = torch.autograd.grad(out, gain, up, retain_graph=True)
    with torch.no_grad():
        gain.add_(1.0)
    got, = torch.autograd.grad(out, gain, up)
    assert torch.equal(got, want)


def test_gains_of_a_frozen_table(cuda):
    for P, K, D in ((1, 1, 1), (300, 9, 48), (300, 9, 129), (20_011, 700, 45)):
        table, codes, s, up = _inputs(P, K, D, torch.float32, seed=P)
        gain = s.clone().requires_grad_(True)
        out = gs.codebook_lookup(table, codes, gain)
        gg, = torch.autograd.grad(out, gain, up)
        _check(table, codes, s, up, out.detach(), None, gg)


@pytest.mark.parametrize("P, K, D", [
    (1, 1, 4), (600, 1, 48), (5000, 3, 7), (16_384, 1, 3), (16_384, 512, 48), (16_001, 500, 129), (14_000, 599, 128),
    (4096, 100_000, 45), (4000, 3000, 200), (4096, 2_200_000, 1), (129, 100_000, 16),
    (40_011, 300, 1), (40_011, 300, 48), (40_011, 2, 513), (16_700, 1, 20), (140_003, 5000, 12), (300_000, 9, 8),
])
@pytest.mark.parametrize("dtype, gain", [(torch.float32, True), (torch.float32, False), (torch.bfloat16, True),
                                         (torch.float16, False)])
@pytest.mark.parametrize("codes", ["most in one", "two blocks", "sorted"])
def test_codes_that_many_rows_have(cuda, P, K, D, dtype, gain, codes):
    """Runs over many chunks and CTAs of the sorted sums, and full queues of the scans.  The longest chain of additions:
    chunks of 16, CTAs of at most 256 chunks, and what a warp of the join takes of 2,501 chunks, below DEPTH."""
    table, c, s, up = _inputs(P, K, D, dtype, torch.int32 if D % 2 else torch.int64, gain, seed=K + D)
    i = torch.arange(P, device="cuda")
    if codes == "most in one":
        c = torch.where(i * 7919 % 10 < 7, K // 2, c)
    elif codes == "two blocks":  # with runs that begin and end anywhere
        c = torch.where(i < P // 3, 0, torch.where(i < P // 3 + 5, -1, K - 1))
    else:
        c = c.sort().values
    args = (table, c.to(torch.int32 if D % 2 else torch.int64), s, up)
    got = _run(*args)
    _check(*args, *got)
    again = _run(*args)
    assert all(torch.equal(x, y) for x, y in zip(got, again) if x is not None)


def test_second_derivatives_and_transforms_are_refused(cuda):
    table, codes, s, up = _inputs(300, 11, 6, torch.float32, seed=7)
    t, gain = table.clone().requires_grad_(True), s.clone().requires_grad_(True)
    want = _run(table, codes, s, up)
    g = torch.autograd.grad(gs.codebook_lookup(t, codes, gain), (t, gain), up.requires_grad_(True), create_graph=True)
    assert torch.equal(g[0].detach(), want[1]) and torch.equal(g[1].detach(), want[2])
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g[0].sum().backward()
    with pytest.raises(RuntimeError, match="functorch"):
        torch.func.grad(lambda x: gs.codebook_lookup(x, codes).sum())(table)


def test_saved_tensors_that_moved(cuda):
    args = _inputs(300, 11, 6, torch.float32, seed=7)
    want = _run(*args)
    with torch.autograd.graph.save_on_cpu():
        t, gain = args[0].clone().requires_grad_(True), args[2].clone().requires_grad_(True)
        out = gs.codebook_lookup(t, args[1], gain)
        got = torch.autograd.grad(out, (t, gain), args[3])
    assert torch.equal(got[0], want[1]) and torch.equal(got[1], want[2])


def test_nothing_to_differentiate_keeps_nothing(cuda):
    table, codes, s, _ = _inputs(300, 11, 6, torch.float32, seed=7)
    assert not gs.codebook_lookup(table, codes, s).requires_grad
    with torch.no_grad():
        assert not gs.codebook_lookup(table.requires_grad_(True), codes, s).requires_grad
    assert gs.codebook_lookup(table, codes, s).requires_grad
    assert gs.codebook_lookup(table.detach(), codes, s.requires_grad_(True)).requires_grad


@pytest.mark.parametrize("D, dtype", [(45, torch.float32), (48, torch.float32), (48, torch.bfloat16)])
@pytest.mark.parametrize("hot", [False, True])
def test_whole_rows_of_a_large_scene(cuda, D, dtype, hot):
    # chunks of 128 rows; a run's 8,594 chunks in CTAs of at least 16 of them: below DEPTH additions
    args = _inputs(1_100_003, 4096, D, dtype, torch.int32, True, seed=D)
    if hot:
        args[1][torch.rand(1_100_003, device="cuda") < 0.6] = 77
    _check(*args, *_run(*args))
