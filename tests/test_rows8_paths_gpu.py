"""The framework's own paths on the operators of act8.py and rownorm.py: layers whose rows are held in 8 bits
(runtime "activations"), and backbones / necks with row norms (norm_cfg type "RMS" | "LN")."""
import os

import pytest
import torch
from torch import nn

from conftest import ROOT

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def full_again(hip_lib):
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from det3d_amd import runtime

    yield
    runtime.configure(activations="full")


def sites(n=1500, shape=(12, 20, 20), c=16, dtype=torch.float32, seed=0):
    from det3d_amd import spconv

    g = torch.Generator().manual_seed(seed)
    d, h, w = shape
    cell = torch.randperm(d * h * w, generator=g)[:n].sort().values
    idx = torch.stack([torch.zeros_like(cell), cell // (h * w), cell // w % h, cell % w], 1).int().cuda()
    feats = torch.randn(n, c, generator=g).to(dtype).cuda()
    return lambda f=None: spconv.SparseConvTensor(feats.clone().requires_grad_() if f is None else f, idx, list(shape), 1)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layer", ["subm 16 32", "strided 32 64", "subm 4 16"])
def test_a_convolution_reads_its_held_rows(layer, dtype, fmt):
    """the output and the data gradient are those of full rows, bit for bit; the weight gradient is act8.weight_grad's"""
    from det3d_amd import act8, runtime, spconv

    kind, cin, cout = layer.split()
    cin, cout = int(cin), int(cout)
    make = sites(c=cin, dtype=dtype)
    conv = (spconv.SubMConv3d(cin, cout, 3, indice_key="a") if kind == "subm" else spconv.SparseConv3d(cin, cout, 3, 2, 1, indice_key="a")).cuda()
    got = {}
    for mode in ("full", fmt):
        runtime.configure(activations=mode)
        x = make()
        y = conv(x)
        dy = torch.randn(y.features.shape, generator=torch.Generator().manual_seed(3)).to(dtype).cuda()
        got[mode] = (y.features.detach(),) + torch.autograd.grad(y.features, [x.features, conv.weight, conv.bias], dy)
    for a, b in zip(got["full"][:2] + got["full"][3:], got[fmt][:2] + got[fmt][3:]):
        assert torch.equal(a, b)
    rb = y.indice_dict["a"]
    rows = nn.functional.pad(x.features.detach(), (0, 16 - cin)) if cin < 16 else x.features.detach()
    want = act8.weight_grad(act8.hold(rows, fmt), dy, rb.nbr_out.view(rb.kvol, rb.cap_out))[:, :cin]
    assert torch.equal(got[fmt][2], want.reshape(conv.weight.shape))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_batch_norm_sweep_reads_its_held_rows(dtype):
    """BatchNorm + ReLU: forward as with full rows; the gradients are the sweeps' at the restored rows and the full rows' statistics"""
    from det3d_amd import act8, runtime, spconv

    torch.manual_seed(0)
    bn = nn.BatchNorm1d(64, eps=1e-3, momentum=0.01).cuda().train()
    with torch.no_grad():
        bn.weight.uniform_(0.5, 1.5)
        bn.bias.normal_()
    x = (torch.randn(900, 64, device="cuda") * 2).to(dtype).requires_grad_()
    dy = torch.randn(900, 64, device="cuda").to(dtype)
    full = spconv.bn_relu(bn, x, True).detach()
    runtime.configure(activations="int8")
    y = spconv.bn_relu(bn, x, True)
    assert torch.equal(y.detach(), full)
    dx, dw, db = torch.autograd.grad(y, [x, bn.weight, bn.bias], dy)
    xr, x64, dy64 = act8.hold(x, "int8").restore().double(), x.detach().double(), dy.double()
    mu, r = x64.mean(0), 1 / torch.sqrt(x64.var(0, unbiased=False) + 1e-3)
    hat = (xr - mu) * r
    pre = hat * bn.weight.detach().double() + bn.bias.detach().double()
    clear = pre.abs() > 1e-4  # (where rounding cannot turn the ReLU's sign; elsewhere the gradient may be either side's)
    assert clear.double().mean() > 0.999
    dz = dy64 * (pre > 0)
    want_b, want_w = dz.sum(0), (dz * hat).sum(0)
    unclear = (dy64.abs() * (1 + hat.abs()) * ~clear).sum(0)
    # 900 float32 additions and a dozen roundings a term
    tol = lambda m: 1000 * 2.0 ** -24 * m + unclear  # noqa: E731
    assert ((db.double() - want_b).abs() <= tol(dz.abs().sum(0))).all()
    assert ((dw.double() - want_w).abs() <= tol((dz * hat).abs().sum(0) + (dz.abs() * (mu.abs() * r + 1)).sum(0))).all()
    want = bn.weight.detach().double() * r * (dz - want_b / 900 - hat * want_w / 900)
    mag = bn.weight.detach().double() * r * (dz.abs() + (dz.abs().sum(0) + unclear) / 900 + (hat.abs() + mu.abs() * r) * ((dz * hat).abs().sum(0) + unclear) / 900)
    slack = bn.weight.detach().double() * r * unclear * (1 + hat.abs()) / 900
    half = 0 if dtype == torch.float32 else 2.0 ** -8
    assert ((dx.double() - want).abs() <= 1000 * 2.0 ** -24 * mag + slack + half * want.abs())[clear].all()


def test_nothing_is_held_without_a_backward_pass(monkeypatch):
    """a model that answers does not pay for the checkpoint, and dense maps keep full rows"""
    from det3d_amd import act8, runtime, spconv

    conv = spconv.SubMConv3d(16, 32, 3, indice_key="a").cuda()
    bn = nn.BatchNorm1d(32, eps=1e-3, momentum=0.01).cuda().train()
    bn2d = nn.BatchNorm2d(32, eps=1e-3, momentum=0.01).cuda().train()
    runtime.configure(activations="int8")
    calls = []
    hold = act8.hold
    monkeypatch.setattr(act8, "hold", lambda *a, **k: calls.append(1) or hold(*a, **k))
    with torch.no_grad():
        want = spconv.bn_relu(bn, conv(sites()()).features, True)
    assert not calls
    assert torch.equal(spconv.bn_relu(bn, conv(sites()()).features, True), want) and len(calls) == 2
    spconv.bn_relu_2d(bn2d, torch.randn(2, 32, 8, 8, device="cuda").contiguous(memory_format=torch.channels_last).requires_grad_(), True)
    assert len(calls) == 2


def _backbone(norm_cfg=None, seed=0):
    from det3d_amd.backbones import SpMiddleResNetFHD

    torch.manual_seed(seed)
    return SpMiddleResNetFHD(num_input_features=5, norm_cfg=norm_cfg).cuda().train()


def _voxels(seed=0, n=4000, batch=2, grid=(64, 96, 41)):
    g = torch.Generator().manual_seed(seed)
    cells = [torch.randperm(grid[2] // 2 * grid[1] * grid[0] // 8, generator=g)[:n // batch].sort().values for _ in range(batch)]
    coors = []
    for b, cell in enumerate(cells):  # a dense corner, so that sites have neighbours
        h, w = grid[1] // 2, grid[0] // 2
        coors.append(torch.stack([torch.full_like(cell, b), cell // (h * w) % grid[2], cell // w % h, cell % w], 1))
    coors = torch.unique(torch.cat(coors), dim=0).int()
    return torch.randn(len(coors), 5, generator=g).cuda(), coors.cuda(), batch, list(grid)


def _step(model, args, seed=1):
    feats, coors, batch, grid = args
    out = model(feats, coors, batch, grid)
    g = torch.randn(out.shape, generator=torch.Generator().manual_seed(seed)).cuda().to(out.dtype)
    grads = torch.autograd.grad(out, [p for p in model.parameters() if p.requires_grad], g)
    return out.detach(), grads


def test_a_backbone_on_held_rows():
    """the whole residual backbone: the same output, gradients a rounding to 8 bits away, less memory between the passes, no bit of
    difference between two runs"""
    from det3d_amd import runtime

    model, args = _backbone(), _voxels()
    out, want = _step(model, args)
    runtime.configure(activations="int8")
    out8, got = _step(model, args)
    _, again = _step(model, args)
    assert torch.allclose(out, out8, rtol=1e-4, atol=1e-4 * float(out.abs().max()))
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    names = [k for k, p in model.named_parameters() if p.requires_grad]
    for k, a, b in zip(names, got, want):
        if k.endswith("weight") and b.dim() == 5:
            # what a rounding to 8 bits changes most is the sign in front of a ReLU.  A pre-activation of deviation 1 in a group
            # whose largest value is 4 is off by at most 4 / 127.5 = 0.031; a share of at most 2 * 0.031 * 0.4 (the normal density
            # at 0) = 0.025 can turn, and one that turns adds or drops its whole gradient: 0.025 of the values against the
            # 0.5 that pass, 0.05 of the gradient's energy a layer.  Over the 21 layers at most 1.05: the cosine between the two
            # gradients is at least 1 / sqrt(1 + 1.05) = 0.70 (that of unrelated ones is near 0)
            cos = float((a * b).sum() / (a.norm() * b.norm()))
            assert cos > 0.70, (k, cos)
    held = {}
    for mode in ("full", "int8"):
        runtime.configure(activations=mode)
        feats, coors, batch, grid = _voxels(1, 60000, 2, (256, 256, 41))
        torch.cuda.synchronize()
        base = torch.cuda.memory_allocated()
        y = model(feats, coors, batch, grid)
        tables = sum(t.numel() * t.element_size() for rb in model.last_indice_dict.values() for t in (rb.nbr_out, rb.nbr_in, rb.dgrad_plan, rb.out_indices) if t is not None)
        held[mode] = torch.cuda.memory_allocated() - base - tables
        del y
    assert held["int8"] < 0.6 * held["full"], held


@pytest.mark.parametrize("kind", ["RMS", "LN"])
def test_a_residual_block_with_row_norms(kind):
    """SparseBasicBlock(norm_cfg = RMS | LN) is conv, norm, ReLU, conv, norm + identity, ReLU: the same convolutions with the norms
    as elementary operations give the same values and gradients"""
    from det3d_amd import spconv
    from det3d_amd.backbones import SparseBasicBlock

    torch.manual_seed(0)
    block = SparseBasicBlock(32, 32, norm_cfg=dict(type=kind, eps=1e-3), indice_key="r").cuda().train()
    make = sites(c=32)

    def plain(m, v):
        if kind == "LN":
            v = v - v.mean(1, keepdim=True)
        v = v / torch.sqrt((v * v).mean(1, keepdim=True) + 1e-3) * m.weight
        return v + m.bias if m.bias is not None else v

    params = list(block.parameters())
    x = make()
    y = block(x).features
    dy = torch.randn(y.shape, generator=torch.Generator().manual_seed(5)).cuda()
    got = torch.autograd.grad(y, [x.features] + params, dy)
    x = make()
    t = block.conv1(x)
    t.features = torch.relu(plain(block.bn1, t.features))
    t = block.conv2(t)
    want_y = torch.relu(x.features + plain(block.bn2, t.features))
    want = torch.autograd.grad(want_y, [x.features] + params, dy)
    assert torch.allclose(y, want_y, rtol=1e-4, atol=1e-4)  # (the convolutions' split products: 2^-16)
    same = (y > 0) == (want_y > 0)
    assert same.all() or (~same).sum() < 10
    for a, b in zip(got, want):
        assert float((a - b).norm()) <= 1e-3 * float(b.norm())


@pytest.mark.parametrize("mode", ["full", "int8"])
@pytest.mark.parametrize("kind", ["RMS", "LN"])
def test_a_backbone_with_row_norms_trains(kind, mode):
    """steps through the whole backbone with row norms (a batch without a site is refused by the planner, as with any norm)"""
    from det3d_amd import runtime

    runtime.configure(activations=mode)
    model, args = _backbone(dict(type=kind, eps=1e-3)), _voxels()
    out, grads = _step(model, args)
    assert torch.isfinite(out).all() and all(torch.isfinite(g).all() and g.any() for g, (k, p) in zip(grads, model.named_parameters()))
    model.eval()
    with torch.no_grad():
        assert torch.allclose(model(*args), out, rtol=1e-4, atol=1e-4 * float(out.abs().max()))  # nothing depends on the mode


@pytest.mark.parametrize("norm_cfg", [None, dict(type="RMS", eps=1e-3)])
def test_a_backbone_on_held_rows_under_autocast(norm_cfg):
    """bfloat16 features all the way: finite gradients of the parameters' type, an output within a bfloat16 pass of the float32 one"""
    from det3d_amd import runtime

    runtime.configure(activations="int8")
    model, args = _backbone(norm_cfg), _voxels()
    with torch.no_grad():
        full = model(*args)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        out, grads = _step(model, args)
    assert out.dtype == torch.bfloat16
    assert all(torch.isfinite(g).all() and g.dtype == p.dtype for g, p in zip(grads, model.parameters()))
    # some 25 layers round their rows to half a step of bfloat16 each, products of them once more: 50 * 2^-8 of the norm at most
    assert float((out.float() - full).norm()) <= 50 * 2.0 ** -8 * float(full.norm())


def test_maps_and_pillars_take_row_norms():
    from det3d_amd.nn_utils import build_norm_layer

    name, m = build_norm_layer(dict(type="LN", eps=1e-3), 24)
    m = m.cuda()
    with torch.no_grad():
        m.weight.normal_()
        m.bias.normal_()
    assert name == "ln" and build_norm_layer(dict(type="RMS"), 8, postfix=2)[0] == "rms2"
    for x in (torch.randn(2, 24, 9, 7, device="cuda"), torch.randn(2, 24, 9, 7, device="cuda").contiguous(memory_format=torch.channels_last),
              torch.randn(5, 24, 11, device="cuda"), torch.randn(6, 24, device="cuda")):
        want = nn.functional.layer_norm(x.movedim(1, -1).double(), (24,), m.weight.double(), m.bias.double(), 1e-3).movedim(-1, 1)
        got = m(x)
        assert got.shape == x.shape and ((got.double() - want).abs() <= 512 * 2.0 ** -24 * (4 + want.abs() * 4)).all()


@pytest.mark.parametrize("mode", ["int8", "e4m3"])
def test_a_detector_trains_on_held_rows(mode):
    """two optimizer steps of the KITTI detector with rows in 8 bits: the first loss is the one of full rows"""
    from det3d_amd import Config, build_detector, runtime, synthetic
    from det3d_amd.trainer import TrainStep

    cfg = Config.fromfile(os.path.join(ROOT, "det3d_amd", "configs", "kitti_car_second.py"))
    dev = torch.device("cuda", 0)
    ds = synthetic.KittiCarSynthetic(n_points=4000, n_seeds=2)
    losses = {}
    for m in ("full", mode):
        runtime.configure(activations=m)
        torch.manual_seed(0)
        model = build_detector(cfg.model, cfg.train_cfg, cfg.test_cfg).to(dev).train()
        step = TrainStep(model, total_steps=10)
        ex = synthetic.make_example(ds.device_batch(0, 2, dev), synthetic.KITTI_CAR)
        losses[m] = [float(step(ex)) for _ in range(2)]
    assert abs(losses[mode][0] - losses["full"][0]) <= 1e-4 * abs(losses["full"][0])
    assert all(v == v and abs(v) < 1e6 for v in losses[mode])


def test_a_table_beyond_the_8_bit_rows_limits():
    """a rulebook with room for more entries than the gradient of held rows can address: the layer keeps full rows, and trains"""
    from det3d_amd import runtime, spconv

    n, kvol, make = 300, 27, sites(n=300, c=16)
    conv = spconv.SubMConv3d(16, 32, 3, indice_key="a").cuda()
    with torch.no_grad():
        rb = conv(make()).indice_dict["a"]
    cap = (1 << 29) // kvol + 1
    table = torch.full((kvol, cap), -1, dtype=torch.int32, device="cuda")
    table[:, :n] = rb.nbr_out.view(kvol, rb.cap_out)[:, :n]
    got = {}
    for mode in ("full", "int8"):
        runtime.configure(activations=mode)
        x = make()
        x.indice_dict["a"] = spconv.Rulebook(kvol, cap, cap, table.view(-1), None, None, n, n, x.indices, rb.out_shape, True)
        y = conv(x).features
        got[mode] = (y.detach(),) + torch.autograd.grad(y, [x.features, conv.weight, conv.bias], torch.ones_like(y))
    assert all(torch.equal(a, b) for a, b in zip(got["full"], got["int8"]))


def test_rows_that_8_bits_do_not_make_smaller(monkeypatch):
    """16 bfloat16 channels are 32 bytes a row, held they are 33: such rows are kept as they are, with the gradients of held ones"""
    from det3d_amd import act8, runtime, spconv
    from det3d_amd.rownorm import RowNorm

    assert not act8.smaller(16, torch.bfloat16) and act8.smaller(24, torch.bfloat16) and act8.smaller(16, torch.float32)
    n, c = 1500, 16
    make = sites(n=n, c=c, dtype=torch.bfloat16)
    torch.manual_seed(0)
    conv = spconv.SubMConv3d(c, 32, 3, indice_key="a").cuda()
    bn = nn.BatchNorm1d(c, eps=1e-3, momentum=0.01).cuda().train()
    norm = RowNorm(c).cuda()
    runtime.configure(activations="int8")

    def step():
        kept, rows = [], make()
        with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t.numel() * t.element_size()) or t, lambda t: t):
            rows.features = spconv.bn_relu(bn, rows.features, True)
            y = conv(rows).features
        params = [conv.weight, bn.weight, bn.bias]
        return [k for k in kept if k % n == 0], torch.autograd.grad(y, params, torch.ones_like(y))

    kept, got = step()
    assert kept == [32 * n] * 2  # (what the sweep and the layer read)
    monkeypatch.setattr(act8, "smaller", lambda *a: True)
    kept, want = step()
    assert kept == [33 * n] * 2
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    monkeypatch.undo()
    x, kept = make().features, []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t.numel() * t.element_size()) or t, lambda t: t):
        norm(x)
    assert max(kept) == 32 * n


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("kind", ["RMS", "LN"])
def test_a_residual_block_with_row_norms_on_held_rows(kind, fmt):
    """the values are those of full rows; every gradient is the formula's at what 8 bits restore of the rows that its layer kept,
    with the ReLUs' signs of the forward pass.  The reference takes the convolutions in full precision mode (split products, 2^-16;
    a dozen of them behind each other, sums no more than ten times their norm: 1e-3) and the norms as float64 formulas"""
    from det3d_amd import act8, rownorm, runtime
    from det3d_amd.backbones import SparseBasicBlock

    torch.manual_seed(0)
    block = SparseBasicBlock(32, 32, norm_cfg=dict(type=kind, eps=1e-3), indice_key="r").cuda().train()
    with torch.no_grad():
        for m in (block.bn1, block.bn2):
            m.weight.uniform_(0.5, 1.5)
    make, params = sites(c=32), list(block.parameters())
    full = block(make()).features.detach()
    runtime.configure(activations=fmt)
    x = make()
    y = block(x).features
    assert torch.equal(y.detach(), full)
    dy = torch.randn(y.shape, generator=torch.Generator().manual_seed(5)).cuda()
    got = torch.autograd.grad(y, [x.features] + params, dy)
    runtime.configure(activations="full")

    def at(v, r):  # the value v with the gradient of r
        return v.detach() + (r - r.detach())

    def restored(v):
        return at(act8.hold(v.detach(), fmt).restore(), v)

    def formula(m, v):
        v = v.double()
        if kind == "LN":
            v = v - v.mean(1, keepdim=True)
        v = v / torch.sqrt((v * v).mean(1, keepdim=True) + 1e-3) * m.weight.double()
        return (v + m.bias.double() if m.bias is not None else v).float()

    def conv(layer, tensor, feats):
        """the layer's output, its data gradient, and the weight gradient at the restored rows"""
        import copy

        still = copy.deepcopy(layer).requires_grad_(False)
        value = tensor.__class__(feats, tensor.indices, tensor.spatial_shape, tensor.batch_size)
        value.indice_dict = tensor.indice_dict
        rows = tensor.__class__(restored(feats).detach(), tensor.indices, tensor.spatial_shape, tensor.batch_size)
        rows.indice_dict = tensor.indice_dict
        r = layer(rows).features
        return still(value).features + (r - r.detach())

    x = make()
    block(x)  # (the rulebook)
    f1 = conv(block.conv1, x, x.features)
    with torch.no_grad():
        n1 = rownorm.norm(f1, block.bn1)
    a = torch.relu(at(n1, formula(block.bn1, restored(f1))))
    f2 = conv(block.conv2, x, a)
    with torch.no_grad():
        h = rownorm.join(x.features, f2, post=block.bn2)
    want_y = torch.relu(at(h, x.features + formula(block.bn2, restored(f2))))
    assert torch.equal(want_y.detach(), full)
    want = torch.autograd.grad(want_y, [x.features] + params, dy)
    for name, g, w in zip(["x"] + [k for k, _ in block.named_parameters()], got, want):
        assert float((g - w).norm()) <= 1e-3 * float(w.norm()), name


@pytest.mark.parametrize("mode,per_value", [("full", 4 + 4 + 4 + 4), ("int8", 3 * 33 / 32 + 4 + 4)])
def test_what_a_residual_block_with_row_norms_keeps(mode, per_value):
    """bytes a value between the passes.  Full: what the first norm and the join read, the first ReLU's output (the second
    convolution's rows too), the second's.  In 8 bits: the rows of the second convolution, the norm and the join, and both ReLUs'
    outputs, which torch keeps as they are; the first convolution's rows belong to the block before"""
    from det3d_amd import act8, runtime
    from det3d_amd.backbones import SparseBasicBlock

    n, c = 60000, 64
    block = SparseBasicBlock(c, c, norm_cfg=dict(type="RMS", eps=1e-3), indice_key="r").cuda().train()
    make = sites(n=n, shape=(30, 60, 60), c=c)
    x = make()
    with torch.no_grad():
        block(x)
    runtime.configure(activations=mode)
    torch.cuda.synchronize()
    base = torch.cuda.memory_allocated()
    y = block(x).features
    kept = torch.cuda.memory_allocated() - base
    kept -= act8.held_bytes(n, c) if mode == "int8" else 0
    assert abs(kept / (n * c) - per_value) < 0.05 * per_value, kept / (n * c)
    del y


@pytest.mark.parametrize("mode", ["full", "int8", "e4m3"])
@pytest.mark.parametrize("shape", [(2, 24, 9, 7), (5, 40, 11)])
def test_gradients_of_row_norms_on_maps(shape, mode):
    """maps in either memory order: the gradients of float64 formulas, under 8 bits those at the restored rows"""
    from det3d_amd import act8, runtime
    from det3d_amd.rownorm import RowNorm

    c = shape[1]
    torch.manual_seed(0)
    m = RowNorm(c, kind="layer").cuda()
    with torch.no_grad():
        m.weight.uniform_(0.5, 1.5)
    runtime.configure(activations=mode)
    v, g = torch.randn(shape, device="cuda"), torch.randn(shape, device="cuda")
    for lay in (lambda t: t, lambda t: t.movedim(1, -1).contiguous().movedim(-1, 1)):
        x = lay(v).clone(memory_format=torch.preserve_format).requires_grad_()
        dx, dw, db = torch.autograd.grad(m(x), [x, m.weight, m.bias], g)
        rows, dz = v.movedim(1, -1).reshape(-1, c), g.movedim(1, -1).reshape(-1, c).double()
        at = (rows if mode == "full" else act8.hold(rows, mode).restore()).double()
        hat = at - at.mean(1, keepdim=True)
        r = 1 / torch.sqrt((hat * hat).mean(1, keepdim=True) + 1e-5)
        hat = hat * r
        d = dz * m.weight.detach().double()
        want = r * (d - d.mean(1, keepdim=True) - hat * (d * hat).mean(1, keepdim=True))
        # (three sums of at most c terms, a dozen roundings, rows of deviation 1 and |hat| <= sqrt(c): 512 steps of the terms' sum)
        mag = r * (d.abs() + d.abs().mean(1, keepdim=True) + (hat.abs() + r) * (d * hat).abs().mean(1, keepdim=True))
        assert ((dx.movedim(1, -1).reshape(-1, c).double() - want).abs() <= 512 * 2.0 ** -24 * mag).all()
        n = rows.shape[0]
        assert ((dw.double() - (dz * hat).sum(0)).abs() <= (512 + 4 * n) * 2.0 ** -24 * (dz.abs() * (hat.abs() + r)).sum(0)).all()
        assert ((db.double() - dz.sum(0)).abs() <= (512 + 4 * n) * 2.0 ** -24 * dz.abs().sum(0)).all()
