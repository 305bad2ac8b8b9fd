"""Workloads of the codebook and class-loss operators, with their plain forms.

Two operators of scene training:

``lookup``  ``scale * table[codes]``: the per-Gaussian rows of an attribute codebook (SH rows, DC colours,
            feature rows), and the gradients of the codebook and of the per-Gaussian gains.
``class``   the softmax cross entropy of a rendered feature map against a label map through a linear
            classifier, and the gradients of the map, the classifier and its bias.

``train`` cases return the outputs and every gradient, the others the outputs alone.
"""

import math

import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # DC colours of a 10,000-Gaussian scene from 256 shared rows: the smallest call, latency counts.
        dict(name="lookup_dc_10k", op="lookup", train=True, P=10_000, K=256, D=3, type="fp32", gain="none",
             index="int64"),
        # One training step of the degree-1..3 SH rows (15 x 3) of a 1M-Gaussian scene; 5% of the Gaussians
        # are not assigned to a row yet.
        dict(name="lookup_shrest_1m", op="lookup", train=True, P=1_000_000, K=4096, D=45, type="fp32", gain="none",
             index="int32", unassigned=0.05),
        # Whole SH rows (16 x 3) of a 6M-Gaussian scene as gain * shape.
        dict(name="lookup_sh_gain_6m", op="lookup", train=True, P=6_000_000, K=16_384, D=48, type="fp32", gain="row",
             index="int32"),
        # Expanding a compressed scene for rendering only: 16-bit rows, an odd number of Gaussians.
        dict(name="lookup_expand_bf16", op="lookup", train=False, P=999_983, K=8192, D=48, type="bf16", gain="row",
             index="int32"),
        # Feature rows of a language-embedded scene in 16 bits, scaled by one factor, an odd row length.
        dict(name="lookup_feature_fp16", op="lookup", train=True, P=300_007, K=50_000, D=77, type="fp16",
             gain="scalar", index="int64"),
        # A 256 x 256 identity map of 16 channels over 256 objects: the small training view.
        dict(name="class_256px", op="class", train=True, layout="map", B=1, H=256, W=256, D=16, V=256, type="fp32",
             bias=True, ignore=0.1, reduction="mean"),
        # The same at 1920 x 1080: the view the renderer is quoted on.
        dict(name="class_1080p", op="class", train=True, layout="map", B=1, H=1080, W=1920, D=16, V=256, type="fp32",
             bias=True, ignore=0.05, reduction="mean"),
        # An 800 x 800 view of 32 channels over 1,000 classes in 16 bits.
        dict(name="class_800px_bf16", op="class", train=True, layout="map", B=1, H=800, W=800, D=32, V=1000,
             type="bf16", bias=False, ignore=0.0, reduction="mean"),
        # Pixels sampled over many views against a large vocabulary of feature codes.
        dict(name="class_sampled_32k", op="class", train=True, layout="rows", N=16_384, D=256, V=32_768, type="bf16",
             bias=True, ignore=0.0, reduction="mean"),
        # A handful of queried pixels against an odd large vocabulary: few rows, a long axis of classes.
        dict(name="class_few_rows", op="class", train=True, layout="rows", N=37, D=128, V=50_001, type="bf16",
             bias=False, ignore=0.0, reduction="sum"),
        # Per-pixel losses of two evaluation views, no gradient.
        dict(name="class_eval_2views", op="class", train=False, layout="map", B=2, H=545, W=979, D=64, V=513,
             type="fp16", bias=True, ignore=0.02, reduction="none"),
        # Full-precision features over a mid-sized vocabulary, odd sizes.
        dict(name="class_fp32_8k", op="class", train=True, layout="rows", N=8191, D=65, V=8200, type="fp32",
             bias=False, ignore=0.3, reduction="sum"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    if rng.random() < 0.4:
        D = rng.choice([1, 2, 3, 12, 27, 45, 48, 64, _log_int(rng, 1, 200)])
        P = _log_int(rng, 1, min(6_000_000, 280_000_000 // D))
        return dict(op="lookup", train=rng.random() < 0.75, P=P, K=_log_int(rng, 1, 100_000), D=D,
                    type=rng.choice(["fp32", "fp32", "bf16", "fp16"]), gain=rng.choice(["none", "scalar", "row"]),
                    index=rng.choice(["int32", "int64"]), unassigned=rng.choice([0.0, 0.0, 0.1, 0.9]))
    kind = rng.choice(["fp32", "bf16", "fp16"])
    D = _log_int(rng, 2, 128 if kind == "fp32" else 256)
    V = _log_int(rng, 2, 65_000)
    cells = 1_000_000_000 if D <= 64 else 300_000_000
    N = _log_int(rng, 1, min(2_000_000, cells // V))
    case = dict(op="class", train=rng.random() < 0.75, D=D, V=V, type=kind, bias=rng.random() < 0.5,
                ignore=rng.choice([0.0, 0.05, 0.6]), reduction=rng.choice(["mean", "mean", "sum", "none"]))
    if rng.random() < 0.5:
        W = max(1, int(math.sqrt(N * rng.uniform(0.5, 2.0))))
        case.update(layout="map", B=rng.choice([1, 1, 2]), H=max(1, N // W // 2), W=W)
    else:
        case.update(layout="rows", N=N)
    return case


def _pixels(case):
    return case["N"] if case["layout"] == "rows" else case["B"] * case["H"] * case["W"]


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dtype = TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device=dev)

    D = case["D"]
    if case["op"] == "lookup":
        P, K = case["P"], case["K"]
        # a few rows are shared by many Gaussians, most by few; which ones is arbitrary
        order = torch.randperm(K, generator=g, device=dev)
        codes = order[(K * uniform(P).double() ** 2).long().clamp_(max=K - 1)]
        if case.get("unassigned", 0.0):
            codes = torch.where(uniform(P) < case["unassigned"], -torch.ones_like(codes), codes)
        codes = codes.to(torch.int32 if case["index"] == "int32" else torch.int64)
        scale = 1.0
        if case["gain"] == "scalar":
            scale = math.sqrt(D)
        elif case["gain"] == "row":
            scale = torch.exp(0.3 * normal(P))
        state = dict(case=case, table=(0.5 * normal(K, D)).to(dtype), codes=codes, scale=scale)
        if case["train"]:
            state["table"].requires_grad_(True)
            if case["gain"] == "row":
                scale.requires_grad_(True)
            # a view's gradient: most Gaussians get a small one, some none
            state["upstream"] = (1e-2 * normal(P, D) * (uniform(P, 1) < 0.8)).to(dtype)
        return state

    V = case["V"]
    weight = normal(V, D) / math.sqrt(D)
    popular = (V * uniform(4096) ** 2).long().clamp_(max=V - 1)
    if case["layout"] == "rows":
        N = case["N"]
        labels = (V * uniform(N) ** 2).long().clamp_(max=V - 1)
        features = 3.0 * weight[labels] + normal(N, D)
    else:
        # segments: a coarse grid of objects, each pixel close to its object's feature
        B, H, W = case["B"], case["H"], case["W"]
        gh, gw = (H + 23) // 24, (W + 31) // 32
        coarse = popular[torch.randint(0, 4096, (B, gh, gw), generator=g, device=dev)]
        labels = coarse.repeat_interleave(24, 1)[:, :H].repeat_interleave(32, 2)[:, :, :W].contiguous()
        features = normal(B, D, H, W)
        features += 3.0 * weight[labels].permute(0, 3, 1, 2)
    if case["ignore"]:
        labels = torch.where(uniform(*labels.shape) < case["ignore"], torch.full_like(labels, -100), labels)
    state = dict(case=case, features=features.to(dtype), weight=weight.to(dtype), labels=labels,
                 bias=0.5 * normal(V) if case["bias"] else None)
    if case["train"]:
        for k in ("features", "weight", "bias"):
            if state[k] is not None:
                state[k].requires_grad_(True)
        state["upstream"] = uniform(*labels.shape) if case["reduction"] == "none" else uniform(())
    return state


def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(state):
    import gswarp_b200 as gs

    case = state["case"]
    if case["op"] == "lookup":
        out = gs.codebook_lookup(state["table"], state["codes"], state["scale"])
        if not case["train"]:
            return {"rows": out}
        leaves = {"table": state["table"]}
        if case["gain"] == "row":
            leaves["scale"] = state["scale"]
        name = "rows"
    else:
        out = gs.class_cross_entropy(state["features"], state["weight"], state["labels"], bias=state["bias"],
                                     reduction=case["reduction"], train=case["train"])
        if not case["train"]:
            return {"loss": out}
        leaves = {k: state[k] for k in ("features", "weight", "bias") if state[k] is not None}
        name = "loss"
    grads = torch.autograd.grad(out, list(leaves.values()), state["upstream"])
    return {name: out.detach(), **dict(zip(("grad_" + k for k in leaves), grads))}


@torch.no_grad()
def _run_plain(state):
    case = state["case"]
    if case["op"] == "lookup":
        table, codes, scale = state["table"], state["codes"].long(), state["scale"]
        used = codes >= 0
        at = codes.clamp(min=0)
        gain = (scale if case["gain"] == "row" else torch.full_like(codes, scale, dtype=torch.float32)) * used
        shape = table.float()[at]
        out = {"rows": (shape * gain[:, None]).to(table.dtype)}
        if case["train"]:
            up = state["upstream"].float()
            total = torch.zeros(table.shape, dtype=torch.float64, device=table.device)
            total.index_add_(0, at, (up * gain[:, None]).double())
            out["grad_table"] = total.to(table.dtype)
            if case["gain"] == "row":
                out["grad_scale"] = (up * shape).sum(1) * used
        return out

    x, w, labels = state["features"].float(), state["weight"].float(), state["labels"]
    rows = x if x.ndim == 2 else x.permute(0, 2, 3, 1).reshape(-1, x.shape[1])
    y = labels.reshape(-1)
    valid = y >= 0
    at = y.clamp(min=0)[:, None]
    z = rows @ w.t()
    if state["bias"] is not None:
        z += state["bias"]
    top = z.max(1, keepdim=True).values
    picked = z.gather(1, at)
    e = (z - top).exp_()
    total = e.sum(1, keepdim=True)
    loss = ((total.log() + top - picked)[:, 0] * valid)
    count = valid.sum().clamp(min=1)
    if case["reduction"] == "none":
        out = {"loss": loss.reshape(labels.shape)}
    else:
        s = loss.double().sum()
        out = {"loss": (s / count if case["reduction"] == "mean" else s).float()}
    if case["train"]:
        up = state["upstream"].reshape(-1) * valid
        if case["reduction"] == "mean":
            up = up / count
        p = e.div_(total)
        p.scatter_add_(1, at, torch.full_like(picked, -1.0))
        p *= up[:, None]
        gx = p @ w
        if x.ndim == 4:
            gx = gx.reshape(x.shape[0], x.shape[2], x.shape[3], x.shape[1]).permute(0, 3, 1, 2).contiguous()
        out["grad_features"] = gx.to(state["features"].dtype)
        out["grad_weight"] = (p.t() @ rows).to(state["weight"].dtype)
        if state["bias"] is not None:
            out["grad_bias"] = p.sum(0)
    return out


@torch.no_grad()
def exact(case, seed):
    """The definitions in 64 bits: sums by sorted segments for the lookup, pieces of rows for the class loss."""
    state = prepare(case, seed)
    if case["op"] == "lookup":
        T, c = state["table"].double(), state["codes"].long()
        s = state["scale"].double() if case["gain"] == "row" else torch.full((len(c),), float(state["scale"]),
                                                                            dtype=torch.float64, device=c.device)
        keep = torch.nonzero(c != -1)[:, 0]
        rows = torch.zeros(len(c), T.shape[1], dtype=torch.float64, device=c.device)
        rows[keep] = T[c[keep]] * s[keep, None]
        out = {"rows": rows}
        if case["train"]:
            g = state["upstream"].double()
            order = keep[torch.argsort(c[keep], stable=True)]
            ends = torch.cumsum(torch.bincount(c[order], minlength=T.shape[0]), 0)
            prefix = torch.zeros(len(order) + 1, T.shape[1], dtype=torch.float64, device=c.device)
            torch.cumsum(g[order] * s[order, None], 0, out=prefix[1:])
            dT = prefix[ends]
            dT[1:] -= prefix[ends[:-1]]
            out["grad_table"] = dT
            if case["gain"] == "row":
                ds = torch.zeros(len(c), dtype=torch.float64, device=c.device)
                ds[keep] = torch.einsum("pd,pd->p", g[keep], T[c[keep]])
                out["grad_scale"] = ds
        return out

    x, W, y = state["features"].double(), state["weight"].double(), state["labels"]
    if x.ndim == 4:
        x = x.movedim(1, -1)
    shape = x.shape
    X, Y = x.reshape(-1, shape[-1]), y.reshape(-1)
    b = state["bias"].double() if state["bias"] is not None else torch.zeros(len(W), dtype=torch.float64,
                                                                             device=W.device)
    n_valid = max(int((Y != -100).sum()), 1)
    losses = torch.zeros(len(X), dtype=torch.float64, device=X.device)
    dX, dW, db = torch.zeros_like(X), torch.zeros_like(W), torch.zeros_like(b)
    piece = max(1, 100_000_000 // len(W))
    for lo in range(0, len(X), piece):
        ids = lo + torch.nonzero(Y[lo:lo + piece] != -100)[:, 0]
        if not len(ids):
            continue
        logp = torch.log_softmax(torch.addmm(b, X[ids], W.T), 1)
        one = torch.arange(len(ids), device=X.device)
        losses[ids] = -logp[one, Y[ids]]
        if case["train"]:
            u = state["upstream"].double()
            u = u.reshape(-1)[ids] if case["reduction"] == "none" else u.expand(len(ids))
            if case["reduction"] == "mean":
                u = u / n_valid
            q = logp.exp()
            q[one, Y[ids]] = torch.expm1(logp[one, Y[ids]])
            q *= u[:, None]
            dX[ids] = q @ W
            dW += q.T @ X[ids]
            db += q.sum(0)
    value = {"none": lambda: losses.reshape(y.shape), "sum": lambda: losses.sum(),
             "mean": lambda: losses.sum() / n_valid}[case["reduction"]]()
    out = {"loss": value}
    if case["train"]:
        dX = dX.reshape(shape)
        out["grad_features"] = dX.movedim(-1, 1).contiguous() if dX.ndim == 4 else dX
        out["grad_weight"] = dW
        if state["bias"] is not None:
            out["grad_bias"] = db
    return out


def work(case):
    size = 4 if case["type"] == "fp32" else 2
    D = case["D"]
    if case["op"] == "lookup":
        P, K = case["P"], case["K"]
        code = 4 if case["index"] == "int32" else 8
        gain = 4 * P if case["gain"] == "row" else 0
        rows, table = P * D * size, K * D * size
        n_bytes = P * code + gain + table + rows
        flops = P * D
        if case["train"]:
            n_bytes += rows + table + gain
            flops += 2 * P * D + (2 * P * D if gain else 0)
        return {"bytes": n_bytes, "flops": flops}
    N, V = _pixels(case), case["V"]
    x, w, b = N * D * size, V * D * size, 4 * V if case["bias"] else 0
    n_bytes = x + w + b + 8 * N + (4 * N if case["reduction"] == "none" else 4)
    flops = 2 * N * V * D + 4 * N * V
    if case["train"]:
        n_bytes += x + w + b + (4 * N if case["reduction"] == "none" else 4)
        flops += 4 * N * V * D + 3 * N * V
    return {"bytes": n_bytes, "flops": flops}
