"""Row norms and the join of a block (det3d_amd/rownorm.py, csrc/d3d_rownorm.hip) on the GPU against float64 formulas and their
differentiation by autograd, over kinds, types, gates, widths, layouts and edges; with rows held in 8 bits; in graphs.

Tolerances: every output has a magnitude M, the formula with absolute values in place of all terms (below, `magnitudes`), and a
float32 evaluation with at most K roundings behind each other is off by at most K 2^-24 M to first order.  A sum over a row passes
at most 8 (in a lane) + 10 (over the lanes) + 16 (over the waves) additions, an output at most three such sums and a dozen products,
each product carrying the errors of both factors: K = 512.  Sums over n rows: K = 512 + 4 n.  Outputs in bfloat16 add half a step, 2^-8."""
import pytest
import torch

pytestmark = pytest.mark.gpu

EPS32 = 2.0 ** -24
HALF = {torch.float32: EPS32, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(scope="module")
def rn(hip_lib):
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from det3d_amd import rownorm as m

    return m


def rand(*shape, seed=0, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed + 17 * sum(shape))) * scale).cuda()


def make(n, c, dtype, gate, seed=0, scale=True, weights=True, bias=True):
    t = {"x": rand(n, c, seed=seed + 1), "f": rand(n, c, seed=seed + 2, scale=3.0) + 0.5, "dh": rand(n, c, seed=seed + 3), "dz": rand(n, c, seed=seed + 4),
         "gate": None if gate is None else rand(n, 1 if gate == "row" else c, seed=seed + 5)}
    t = {k: None if v is None else v.to(dtype) for k, v in t.items()}
    t["scale"] = rand(c, seed=seed + 6) if scale else None
    for k, i in (("post_w", 7), ("pre_w", 8)):
        t[k] = 1 + rand(c, seed=seed + i, scale=0.3) if weights else None
    for k, i in (("post_b", 9), ("pre_b", 10)):
        t[k] = rand(c, seed=seed + i, scale=0.3) if bias else None
    return t


LEAVES = ("x", "f", "gate", "scale", "post_w", "post_b", "pre_w", "pre_b")


def hat_of(v, kind, eps):
    m = v.mean(1, keepdim=True) if kind == "layer" else 0.0
    r = 1 / torch.sqrt(((v - m) ** 2).mean(1, keepdim=True) + eps)
    return (v - m) * r, r


def act_of(g, act):
    return {"none": lambda: g, "sigmoid": lambda: torch.sigmoid(g), "silu": lambda: g * torch.sigmoid(g)}[act]()


def forward64(t, post, pre, act, alpha, eps):
    out = {}
    h = t["x"]
    if t.get("f") is not None:
        u = t["f"]
        if post:
            u, _ = hat_of(u, post, eps)
            u = u * t["post_w"] if t["post_w"] is not None else u
            u = u + t["post_b"] if t["post_b"] is not None else u
        if t["scale"] is not None:
            u = u * t["scale"]
        if t["gate"] is not None:
            u = u * act_of(t["gate"], act)
        h = h + alpha * u
        out["h"] = h
    if pre:
        z, _ = hat_of(h, pre, eps)
        z = z * t["pre_w"] if t["pre_w"] is not None else z
        out["z"] = z + t["pre_b"] if t["pre_b"] is not None else z
    return out


def magnitudes(t, post, pre, act, alpha, eps):
    """M of every output (see above)"""
    one = torch.ones((), dtype=torch.float64)
    ab = lambda k: t[k].abs() if t.get(k) is not None else None  # noqa: E731
    has_f = t.get("f") is not None

    def hat_m(v, mv, kind):  # of the normalised rows, r, and 1 + the relative error of r
        hat, r = hat_of(v, kind, eps)
        rel = (hat.abs() * r * mv).mean(1, keepdim=True)
        return hat.abs() + r * (mv + (mv.mean(1, keepdim=True) if kind == "layer" else 0)) + hat.abs() * rel, r, 1 + rel

    M = {}
    h, mh = t["x"], t["x"].abs()
    mfh = mu = None
    fr = frho = one
    if has_f:
        mfh = t["f"].abs()
        if post:
            mfh, fr, frho = hat_m(t["f"], t["f"].abs(), post)
        mu = mfh * (ab("post_w") if t["post_w"] is not None else one) + (ab("post_b") if t["post_b"] is not None else 0)
        g = t["gate"]
        ma = one if g is None else (act_of(g, act).abs() + (g.abs() * 0.25 if act != "none" else 0))  # (the slope times g's own error)
        sa = abs(alpha) * (ab("scale") if t["scale"] is not None else one)
        h = forward64(t, post, None, act, alpha, eps)["h"]
        mh = mh + sa * ma * mu
        M["h"] = mh
    mhh, hr, hrho = (mh, one, one) if not pre else hat_m(h, mh, pre)
    dz = ab("dz") if pre else None
    if pre:
        w = ab("pre_w") if t["pre_w"] is not None else one
        M["z"] = mhh * w + (ab("pre_b") if t["pre_b"] is not None else 0)
        d = dz * w
        md = hr * hrho * (d + d.mean(1, keepdim=True) + mhh * (d * mhh).mean(1, keepdim=True))
        M["pre_w"], M["pre_b"] = (dz * mhh).sum(0), dz.sum(0)
    else:
        md = torch.zeros_like(mh)
    if has_f:
        md = md + ab("dh")
    M["x"] = md
    if has_f:
        mdu = sa * ma * md
        d = mdu * (ab("post_w") if t["post_w"] is not None else one)
        M["f"] = d if not post else fr * frho * (d + d.mean(1, keepdim=True) + mfh * (d * mfh).mean(1, keepdim=True))
        M["post_w"], M["post_b"] = (mdu * mfh).sum(0), mdu.sum(0)
        M["scale"] = (abs(alpha) * ma * md * mu).sum(0)
        if g is not None:
            slope = one if act == "none" else 1.1 + g.abs() * 0.25
            mg = sa * md * mu * slope
            M["gate"] = mg if g.shape[1] == t["x"].shape[1] else mg.sum(1, keepdim=True)
    return M


def run(rn, t, post, pre, act, alpha, eps, checkpoint=None, use_h=True, use_z=True):
    """outputs and gradients of the framework's call"""
    leaf = {k: t[k].detach().clone().requires_grad_() for k in LEAVES if t.get(k) is not None}
    g = leaf.get
    pre_s = rn.NormSpec(pre, g("pre_w"), g("pre_b"), eps) if pre else None
    if t.get("f") is None:
        outs = {"z": rn.norm(leaf["x"], pre_s, checkpoint=checkpoint)}
    else:
        post_s = rn.NormSpec(post, g("post_w"), g("post_b"), eps) if post else None
        o = rn.join(leaf["x"], leaf["f"], post=post_s, pre=pre_s, gate=g("gate"), gate_act=act, scale=g("scale"), alpha=alpha, checkpoint=checkpoint)
        outs = {"h": o[0], "z": o[1]} if pre else {"h": o}
    ends = [(v, t["d" + k]) for k, v in outs.items() if (k == "h" and use_h) or (k == "z" and use_z)]
    used = list(leaf)
    if not pre:
        used = [k for k in used if not k.startswith("pre")]
    if not post:
        used = [k for k in used if not k.startswith("post")]
    grads = torch.autograd.grad([e[0] for e in ends], [leaf[k] for k in used], [e[1] for e in ends], allow_unused=True)
    return {k: v.detach() for k, v in outs.items()}, dict(zip(used, grads))


def check(rn, t, post, pre, act="none", alpha=1.0, eps=1e-5, checkpoint=None, at=None):
    """`at`: the rows where the gradients are taken (restored x and f), default t's own"""
    outs, grads = run(rn, t, post, pre, act, alpha, eps, checkpoint)
    n, c = t["x"].shape
    dtype = t["x"].dtype
    d64 = lambda s: {k: v.detach().cpu().double() if v is not None else None for k, v in s.items()}  # noqa: E731
    t64 = d64(t)
    want, M = forward64(t64, post, pre, act, alpha, eps), magnitudes(t64, post, pre, act, alpha, eps)
    for k, v in outs.items():
        assert v.dtype == dtype and v.shape == (n, c)
        off = (v.cpu().double() - want[k]).abs()
        tol = 512 * EPS32 * M[k] + (HALF[dtype] * want[k].abs() if dtype != torch.float32 else 0)
        assert (off <= tol).all(), (k, float((off - tol).max()))
    t64 = d64({**t, **(at or {})})
    leaf = {k: v.requires_grad_() if k in LEAVES and v is not None else v for k, v in t64.items()}
    w = forward64(leaf, post, pre, act, alpha, eps)
    total = sum((v * t64["d" + k]).sum() for k, v in w.items())
    names = list(grads)
    want = dict(zip(names, torch.autograd.grad(total, [leaf[k] for k in names])))
    with torch.no_grad():
        M = magnitudes({k: v.detach() if v is not None else None for k, v in leaf.items()}, post, pre, act, alpha, eps)
    for k in names:
        got = grads[k]
        rows = k in ("x", "f", "gate")
        assert got.dtype == (dtype if rows else torch.float32) and got.shape == want[k].shape, k
        tol = (512 if rows else 512 + 4 * n) * EPS32 * M[k]
        if k == "gate" and t["gate"].shape[1] == 1 and c > 1:
            tol = 1024 * EPS32 * M[k]
        if rows and dtype != torch.float32:
            tol = tol + HALF[dtype] * want[k].abs()
        off = (got.cpu().double() - want[k]).abs()
        assert (off <= tol + 1e-300).all(), (k, float((off - tol).max()), float(M[k].max()))
    return outs, grads


DTYPES = [torch.float32, torch.bfloat16]
KINDS = ["rms", "layer"]
SIZES = [(1, 1), (1, 16), (3, 5), (17, 16), (9, 32), (50, 64), (21, 100), (12, 128), (40, 130), (7, 256), (5, 333), (6, 520), (4, 1000),
         (3, 1024), (2, 2048), (3, 2500), (2, 4096), (2, 8191), (3, 8192), (700, 24)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,c", SIZES)
def test_norm(rn, n, c, dtype, kind):
    t = {k: v for k, v in make(n, c, dtype, None).items() if k in ("x", "dz", "pre_w", "pre_b")}
    t.update(f=None, scale=None, gate=None, post_w=None, post_b=None)
    check(rn, t, None, kind)


@pytest.mark.parametrize("gate,act", [(None, "none"), ("row", "sigmoid"), ("full", "silu"), ("full", "none")])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,c", SIZES)
def test_join(rn, n, c, dtype, gate, act):
    check(rn, make(n, c, dtype, gate), "rms", "rms" if n % 2 else "layer", act, alpha=0.5)


@pytest.mark.parametrize("post,pre", [("rms", "layer"), ("layer", "rms"), ("layer", None), (None, "rms"), (None, None)])
@pytest.mark.parametrize("gate,act", [(None, "none"), ("row", "silu"), ("full", "sigmoid"), ("row", "none")])
@pytest.mark.parametrize("vectors", ["all", "no bias", "none"])
def test_absent_parts(rn, post, pre, gate, act, vectors):
    t = make(37, 48, torch.float32, gate, scale=vectors != "none", weights=vectors != "none", bias=vectors == "all")
    check(rn, t, post, pre, act, alpha=1.0 if vectors == "all" else -0.25)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,c", [(1, 1), (5, 16), (33, 20), (20, 64), (9, 100), (4, 333), (3, 1024), (2, 4096), (2, 8191), (300, 128)])
def test_gradients_at_the_held_rows(rn, n, c, dtype, fmt):
    """held in 8 bits: the forward pass is the one of the rows, the backward pass bit for bit the one at the restored rows"""
    from det3d_amd import act8

    t = make(n, c, dtype, "full")
    at = {k: act8.hold(t[k], fmt).restore() for k in ("x", "f")}
    outs, grads = check(rn, t, "rms", "layer", "sigmoid", 0.5, checkpoint=fmt, at=at)
    plain_outs, _ = run(rn, t, "rms", "layer", "sigmoid", 0.5, 1e-5)
    _, want = run(rn, {**t, **at}, "rms", "layer", "sigmoid", 0.5, 1e-5)
    assert all(torch.equal(outs[k], plain_outs[k]) for k in outs)
    assert all(torch.equal(grads[k], want[k]) for k in grads)


@pytest.mark.parametrize("use_h,use_z", [(True, False), (False, True)])
def test_one_of_the_two_outputs_alone(rn, use_h, use_z):
    t = make(30, 64, torch.float32, "full")
    _, got = run(rn, t, "rms", "rms", "sigmoid", 0.5, 1e-5, use_h=use_h, use_z=use_z)
    zero = {"dh": t["dh"] * use_h, "dz": t["dz"] * use_z}
    _, want = run(rn, {**t, **zero}, "rms", "rms", "sigmoid", 0.5, 1e-5)
    for k in got:
        assert torch.equal(got[k] if got[k] is not None else torch.zeros_like(want[k]), want[k]), k


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(rn, dtype):
    """rows at a distance, unaligned starts, transposed and expanded operands give what contiguous ones give"""
    big = {k: rand(140, 90, seed=i).to(dtype) for i, k in enumerate(("x", "f", "gate", "dh", "dz"))}
    w = make(1, 64, dtype, None)
    for cut in (lambda a: a[:50, :64], lambda a: a[2:52, 3:67], lambda a: a[::2, 8:72][:50], lambda a: a.t()[:50, :64],
                lambda a: a[:1, :64].expand(50, 64)):
        t = {**w, **{k: cut(v) for k, v in big.items()}}
        outs, grads = [], []
        for tt in (t, {k: v.contiguous() if v is not None else None for k, v in t.items()}):
            leaf = {k: tt[k].detach().requires_grad_() for k in LEAVES}
            h, z = rn.join(leaf["x"], leaf["f"], post=rn.NormSpec("rms", leaf["post_w"], leaf["post_b"], 1e-5),
                           pre=rn.NormSpec("layer", leaf["pre_w"], leaf["pre_b"], 1e-5), gate=leaf["gate"], gate_act="sigmoid", scale=leaf["scale"])
            outs.append((h, z))
            grads.append(torch.autograd.grad((h, z), list(leaf.values()), (tt["dh"], tt["dz"])))
        # (unaligned rows are summed in another order: a few roundings apart)
        for a, b in zip(outs[0] + grads[0], outs[1] + grads[1]):
            assert (a - b).abs().max() <= (2 * HALF[dtype] + 1024 * EPS32) * max(1.0, float(b.detach().abs().max())), dtype


def test_gradients_by_differences(rn):
    """the gradient is the slope: along a random direction, central differences of float64 formulas at the float32 point"""
    t = make(11, 40, torch.float32, "full")
    _, grads = run(rn, t, "layer", "rms", "silu", 0.5, 1e-5)
    t64 = {k: v.cpu().double() if v is not None else None for k, v in t.items()}

    def loss(step):
        s = {k: v + step * rand(*v.shape, seed=99).cpu().double() if k in LEAVES else v for k, v in t64.items()}
        return sum((v * t64["d" + k]).sum() for k, v in forward64(s, "layer", "rms", "silu", 0.5, 1e-5).items())

    slope = float(loss(1e-5) - loss(-1e-5)) / 2e-5
    got = sum(float((g.cpu().double() * rand(*g.shape, seed=99).cpu().double()).sum()) for g in grads.values())
    scale = sum(float((g.cpu().double() * rand(*g.shape, seed=99).cpu().double()).abs().sum()) for g in grads.values())
    assert abs(got - slope) <= 1e-6 * scale  # differences: 1e-10 relative curvature and 1e-16 / 1e-5; float32 sums: below 512 2^-24


def test_rows_stay_by_themselves(rn):
    """a row of NaN, infinities or zeros changes no other row; no row at all"""
    t = make(9, 64, torch.float32, "full")
    spec = rn.NormSpec("layer", t["pre_w"], t["pre_b"], 1e-5)
    post = rn.NormSpec("rms", t["post_w"], t["post_b"], 1e-5)
    h0, z0 = rn.join(t["x"], t["f"], post=post, pre=spec, gate=t["gate"], gate_act="sigmoid", scale=t["scale"])
    x, f = t["x"].clone(), t["f"].clone()
    x[2], f[5, 3], f[7] = float("nan"), float("inf"), 0
    h1, z1 = rn.join(x, f, post=post, pre=spec, gate=t["gate"], gate_act="sigmoid", scale=t["scale"])
    same = [0, 1, 3, 4, 6, 8]
    assert torch.equal(h0[same], h1[same]) and torch.equal(z0[same], z1[same])
    assert torch.isnan(z1[2]).all() and torch.isnan(z1[5]).any() and torch.isfinite(z1[7]).all()
    leaf = {k: (t[k][:0] if t[k].dim() == 2 else t[k]).clone().requires_grad_() for k in LEAVES}
    h, z = rn.join(leaf["x"], leaf["f"], post=rn.NormSpec("rms", leaf["post_w"], leaf["post_b"], 1e-5),
                   pre=rn.NormSpec("rms", leaf["pre_w"], leaf["pre_b"], 1e-5), gate=leaf["gate"], scale=leaf["scale"], checkpoint="int8")
    grads = torch.autograd.grad((h, z), list(leaf.values()), (t["dh"][:0], t["dz"][:0]))
    assert h.shape == (0, 64) and not any(g.any() for g in grads)


def test_wide_sums_are_the_same_twice(rn):
    t = make(3000, 96, torch.bfloat16, "row")
    a, ga = run(rn, t, "rms", "layer", "sigmoid", 0.5, 1e-5, "int8")
    b, gb = run(rn, t, "rms", "layer", "sigmoid", 0.5, 1e-5, "int8")
    assert all(torch.equal(a[k], b[k]) for k in a) and all(torch.equal(ga[k], gb[k]) for k in ga)


@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_in_a_graph_and_on_another_stream(rn, checkpoint):
    t = make(400, 64, torch.float32, "row")
    leaf = {k: t[k].clone().requires_grad_() for k in LEAVES}

    def step():
        h, z = rn.join(leaf["x"], leaf["f"], post=rn.NormSpec("rms", leaf["post_w"], leaf["post_b"], 1e-5),
                       pre=rn.NormSpec("layer", leaf["pre_w"], leaf["pre_b"], 1e-5), gate=leaf["gate"], gate_act="sigmoid",
                       scale=leaf["scale"], checkpoint=checkpoint)
        return (h.detach(), z.detach()) + torch.autograd.grad((h, z), list(leaf.values()), (t["dh"], t["dz"]))

    want = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del got, want
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for k in range(3):
        with torch.no_grad():
            leaf["x"].copy_(rand(400, 64, seed=50 + k))
            leaf["f"].copy_(rand(400, 64, seed=60 + k))
        want = step()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_saved_tensors_that_were_packed_away(rn, checkpoint):
    """hooks that move what is saved for the backward pass (to the host and back): the same gradients"""
    t = make(300, 72, torch.float32, "row")
    leaf = {k: t[k].clone().requires_grad_() for k in LEAVES}

    def step():
        h, z = rn.join(leaf["x"] * 1.0, leaf["f"] * 1.0, post=rn.NormSpec("rms", leaf["post_w"], leaf["post_b"], 1e-5),
                       pre=rn.NormSpec("layer", leaf["pre_w"], leaf["pre_b"], 1e-5), gate=leaf["gate"], gate_act="silu",
                       scale=leaf["scale"], checkpoint=checkpoint)
        return lambda: torch.autograd.grad((h, z), list(leaf.values()), (t["dh"], t["dz"]))

    want = step()()
    with torch.autograd.graph.save_on_cpu():
        later = step()
    keep = [torch.full((300, 72), float("nan"), device="cuda") for _ in range(8)]  # (where the packed tensors lay)
    got = later()
    assert len(keep) == 8 and all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("c,dtype", [(4096, torch.bfloat16), (8192, torch.bfloat16), (8192, torch.float32), (4093, torch.bfloat16)])
def test_wide_rows_in_a_graph_and_two_at_once(rn, c, dtype):
    """rows whose [c] vectors take most of a CU's LDS: a first call that is captured, and two streams at the same time"""
    t = make(21, c, dtype, "full")
    leaf = {k: t[k].clone().requires_grad_() for k in LEAVES}

    def step():
        h, z = rn.join(leaf["x"], leaf["f"], post=rn.NormSpec("rms", leaf["post_w"], leaf["post_b"], 1e-5),
                       pre=rn.NormSpec("layer", leaf["pre_w"], leaf["pre_b"], 1e-5), gate=leaf["gate"], gate_act="silu",
                       scale=leaf["scale"], checkpoint="e4m3")
        return (h.detach(), z.detach()) + torch.autograd.grad((h, z), list(leaf.values()), (t["dh"], t["dz"]))

    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    want = step()
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    streams = [torch.cuda.Stream() for _ in range(2)]
    both = [[], []]
    for _ in range(3):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                both[k].append(step())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for k in range(2) for r in both[k] for a, b in zip(r, want))


def test_refusals(rn):
    from det3d_amd._lib import D3dError

    t = make(6, 32, torch.float32, "full")
    spec = rn.NormSpec("rms", t["pre_w"], None, 1e-5)
    x, f = t["x"], t["f"]
    for bad, match in ((lambda: rn.norm(x.half(), spec), "float32 / bfloat16"), (lambda: rn.norm(x.cpu(), spec), "GPU only"),
                       (lambda: rn.norm(x[0], spec), "rows"), (lambda: rn.norm(x[:, :31], spec), "weight"),
                       (lambda: rn.norm(x, spec._replace(weight=t["pre_w"].bfloat16())), "weight"),
                       (lambda: rn.norm(torch.zeros(2, 8193, device="cuda"), spec), "at most 8192"),
                       (lambda: rn.join(x, f.bfloat16(), pre=spec), "bfloat16"), (lambda: rn.join(x, f[:5], pre=spec), "and f"),
                       (lambda: rn.join(x, f, pre=spec, gate=t["gate"][:, :4]), "gate"), (lambda: rn.join(x, f, pre=spec, scale=t["scale"][:4]), "scale")):
        with pytest.raises(D3dError, match=match):
            bad()
    for bad, match in ((lambda: rn.norm(x, spec._replace(kind="batch")), "kind"), (lambda: rn.norm(x, spec._replace(eps=-1.0)), "eps"),
                       (lambda: rn.norm(x, spec, checkpoint="fp4"), "format"), (lambda: rn.norm(x, None), "no norm"),
                       (lambda: rn.join(x, f, gate=t["gate"], gate_act="relu"), "gate_act"), (lambda: rn.join(x, f, gate_act="silu"), "without a gate")):
        with pytest.raises(ValueError, match=match):
            bad()
    leaf = x.clone().requires_grad_()
    with pytest.raises(D3dError, match="create_graph"):  # no second derivatives, rather than wrong ones
        torch.autograd.grad(rn.norm(leaf, spec).sum(), leaf, create_graph=True)


@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
def test_strided_rows_that_were_packed_away(rn, checkpoint):
    """x, f and gate as halves of wider rows that are freed once they are packed: the copies that come back may lie where those lay"""
    t = make(200, 64, torch.float32, "full")
    names = ("x", "f", "gate")

    def step(pack):
        leaf = {k: v.clone().requires_grad_() for k, v in t.items() if k in LEAVES}
        half = {k: torch.cat([leaf[k], leaf[k]], 1)[:, :64] for k in names}  # rows 128 apart, nobody else's
        with pack:
            h, z = rn.join(half["x"], half["f"], post=rn.NormSpec("rms", leaf["post_w"], leaf["post_b"], 1e-5),
                           pre=rn.NormSpec("layer", leaf["pre_w"], leaf["pre_b"], 1e-5), gate=half["gate"], gate_act="silu",
                           scale=leaf["scale"], checkpoint=checkpoint)
        del half
        return torch.autograd.grad((h, z), list(leaf.values()), (t["dh"], t["dz"]))

    import contextlib

    want = step(contextlib.nullcontext())
    for _ in range(3):
        got = step(torch.autograd.graph.save_on_cpu())
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("fmt", [None, "int8", "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gate,act", [(None, "none"), ("row", "sigmoid"), ("full", "silu")])
@pytest.mark.parametrize("n,c", [(1, 1), (7, 16), (40, 130), (5, 333), (300, 64), (3, 2500), (2, 8192)])
def test_a_join_without_a_pre_norm(rn, n, c, gate, act, dtype, fmt):
    """the residual block's join: its gradients are those at f (held: at the restored f), whatever x was"""
    from det3d_amd import act8

    t = make(n, c, dtype, gate)
    at = None if fmt is None else {"f": act8.hold(t["f"], fmt).restore()}
    _, grads = check(rn, t, "layer" if n % 2 else "rms", None, act, alpha=0.5, checkpoint=fmt, at=at)
    assert torch.equal(grads["x"], t["dh"])
    _, other = run(rn, {**t, "x": torch.full_like(t["x"], float("inf"))}, "layer" if n % 2 else "rms", None, act, 0.5, 1e-5, fmt)
    assert all(torch.equal(grads[k], other[k]) for k in grads)


@pytest.mark.parametrize("fmt", [None, "int8"])
@pytest.mark.parametrize("pre", [False, True])
def test_what_a_join_keeps(rn, fmt, pre):
    """bytes between the passes: h (and z), f, and x only where a pre norm's backward pass reads it"""
    from det3d_amd import act8

    n, c = 40000, 64
    x, f = rand(n, c, seed=1).requires_grad_(), rand(n, c, seed=2).requires_grad_()
    spec = rn.NormSpec("rms", None, None, 1e-5)
    full, held = 4 * n * c, act8.held_bytes(n, c)
    torch.cuda.synchronize()
    base = torch.cuda.memory_allocated()
    out = rn.join(x * 1, f * 1, post=spec, pre=spec if pre else None, checkpoint=fmt)
    kept = torch.cuda.memory_allocated() - base
    want = full * (2 if pre else 1) + (held if fmt else full) * (2 if pre else 1)
    assert want <= kept <= want + 4 * (1 << 21), (kept, want)  # (the allocator's blocks: 2 MiB each)
    del out


def test_activations_far_from_zero(rn):
    """sigmoid, SiLU and their slopes by relative error.  With u = 2^-24: the exponent -g log2 e is rounded twice (1.25 u of it, with the
    constant's own error), which is 1.25 |g| u of the exponential; that and the reciprocal are a step (2 u) off, the sum u: p by
    (1.25 |g| + 5) u.  SiLU adds a product.  Slopes: p - p p, off by p's error and 2 u where p is small, 5 u in all where it is near 1"""
    g = torch.cat([torch.linspace(-85, 85, 4097), torch.tensor([-80.0, -50.0, -20.0, -10.0, -1e-3, 0.0, 1e-30, 20.0])]).cuda()
    n = g.numel()
    one, zero = torch.ones(n, 1, device="cuda"), torch.zeros(n, 1, device="cuda")
    # (two channels with the same gate: a full gate, h = act(g) exactly)
    f, x = one.expand(n, 2).contiguous(), zero.expand(n, 2).contiguous()
    g64 = g.cpu().double()
    p = 1 / (1 + torch.exp(-g64))
    rel = (1.25 * g64.abs() + 5) * EPS32
    for act, want, slope in (("sigmoid", p, p * (1 / (1 + torch.exp(g64)))), ("silu", g64 * p, p * (1 + g64 / (1 + torch.exp(g64))))):
        gate = g[:, None].expand(n, 2).contiguous().requires_grad_()
        h = rn.join(x, f, gate=gate, gate_act=act)
        off = (h.detach()[:, 1].cpu().double() - want).abs()
        assert (off <= (rel + (act == "silu") * EPS32) * want.abs()).all(), (act, float((off / want.abs().clamp(min=1e-300) / EPS32).max()))
        (dg,) = torch.autograd.grad(h, gate, torch.ones_like(h))
        off = (dg[:, 0].cpu().double() - slope).abs()
        if act == "sigmoid":
            tol = (rel + 2 * EPS32) * slope + 5 * EPS32 * (g64 > 0)
        else:  # p + a (1 - p): both terms by p's error, the second with |g|'s weight, three roundings
            tol = (rel + 3 * EPS32) * (p + g64.abs() * p / (1 + torch.exp(g64))) + 5 * EPS32 * g64.abs() * p * (g64 > 0)
        assert (off <= tol).all(), (act, float(((off - tol) / EPS32).max()))
    far = torch.tensor([[-1e30, -1e30], [-100.0, -88.0], [100.0, 1e30], [float("inf"), float("-inf")]], device="cuda")
    h = rn.join(torch.zeros_like(far), torch.ones_like(far), gate=far, gate_act="sigmoid").cpu()
    assert (h[:2] <= 2.0 ** -126).all() and (h[:2] >= 0).all() and (h[2] == 1).all() and h[3].tolist() == [1.0, 0.0]


@pytest.mark.parametrize("checkpoint", [None, "int8"])
@pytest.mark.parametrize("pre", [None, "layer"])
def test_one_tensor_in_every_place_and_two_backward_passes(rn, pre, checkpoint):
    """x, f and gate are the same rows, the output's gradient is expanded from one number, the graph is gone through twice"""
    from det3d_amd import act8

    n, c = 50, 64
    v, w = rand(n, c, seed=3), 1 + rand(c, seed=4, scale=0.3)
    leaf, weight = v.clone().requires_grad_(), w.clone().requires_grad_()
    post, pre_s = rn.NormSpec("rms", weight, None, 1e-5), rn.NormSpec(pre, weight, None, 1e-5) if pre else None
    out = rn.join(leaf, leaf, post=post, pre=pre_s, gate=leaf, gate_act="sigmoid", checkpoint=checkpoint)
    total = out[0].sum() + 2 * out[1].sum() if pre else out.sum()
    first = torch.autograd.grad(total, [leaf, weight], retain_graph=True)
    second = torch.autograd.grad(total, [leaf, weight])
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    # the definition: x and f at the rows that the checkpoint restores, the gate as it came
    at = act8.hold(v, checkpoint).restore() if checkpoint else v
    one = torch.ones(n, c, device="cuda")
    t = {"x": at, "f": at, "gate": v, "scale": None, "post_w": w, "post_b": None, "pre_w": w if pre else None, "pre_b": None, "dh": one, "dz": 2 * one}
    d64 = {k: a.cpu().double() if a is not None else None for k, a in t.items()}
    l64 = {k: a.clone().requires_grad_() if k in LEAVES and a is not None else a for k, a in d64.items()}
    ends = forward64(l64, "rms", pre, "sigmoid", 1.0, 1e-5)
    names = [k for k in LEAVES if l64.get(k) is not None]
    want = dict(zip(names, torch.autograd.grad(sum((e * d64["d" + k]).sum() for k, e in ends.items()), [l64[k] for k in names])))
    M = magnitudes(d64, "rms", pre, "sigmoid", 1.0, 1e-5)
    for got, parts, k in ((first[0], ("x", "f", "gate"), 512 + 3), (first[1], ("post_w", "pre_w") if pre else ("post_w",), 512 + 4 * n + 2)):
        off = (got.cpu().double() - sum(want[p] for p in parts)).abs()
        tol = k * EPS32 * sum(M[p] for p in parts)
        assert (off <= tol).all(), float((off - tol).max())
