"""Argument checks of the operators on held rows and row norms (d3d_act8_*, d3d_row_join_*): they run before any HIP call, so no GPU
is needed; what the Python layer refuses without one; workspace sizes."""
import ctypes

import pytest
import torch


def err(L):
    return L.d3d_last_error()


def test_pitch_and_workspaces(hip_lib):
    L = hip_lib
    assert [L.d3d_act8_pitch(c) for c in (1, 31, 32, 33, 64, 4096)] == [32, 32, 32, 64, 64, 4096]
    assert L.d3d_act8_pitch(0) == 0 and L.d3d_act8_pitch(-3) == 0
    from det3d_amd import act8

    assert all(act8.pitch(c) == L.d3d_act8_pitch(c) for c in range(1, 300))
    assert L.d3d_act8_wgrad_workspace_bytes(0, 27, 64, 64, 0) == 0 and L.d3d_act8_wgrad_workspace_bytes(100, 27, 64, 64, 9) == 0
    big = L.d3d_act8_wgrad_workspace_bytes(100000, 27, 64, 64, 0)
    assert big % (27 * 64 * 64 * 4) == 0 and big < 1 << 30
    assert L.d3d_row_join_ws_floats(100, 64, 0, 5) >= 5 * 64
    for bad in ((0, 64, 0, 5), (100, 0, 0, 5), (100, 8193, 0, 5), (100, 64, 2, 5), (100, 64, 0, 0), (100, 64, 0, 6)):
        assert L.d3d_row_join_ws_floats(*bad) == 0


def test_hold_and_restore_refuse(hip_lib):
    L = hip_lib
    assert L.d3d_act8_hold(1, 64, 10, 64, 7, 0, 16, 1, None) == -1 and b"dtype" in err(L)
    assert L.d3d_act8_hold(1, 64, 10, 64, 0, 2, 16, 1, None) == -1 and b"format" in err(L)
    assert L.d3d_act8_hold(1, 64, -1, 64, 0, 0, 16, 1, None) == -1 and b"rows" in err(L)
    assert L.d3d_act8_hold(1, 64, 10, 0, 0, 0, 16, 1, None) == -1
    assert L.d3d_act8_hold(1, 63, 10, 64, 0, 0, 16, 1, None) == -1 and b"apart" in err(L)
    assert L.d3d_act8_hold(None, 64, 10, 64, 0, 0, 16, 1, None) == -1 and b"null" in err(L)
    assert L.d3d_act8_hold(1, 64, 10, 64, 0, 0, 8, 1, None) == -1 and b"aligned" in err(L)
    assert L.d3d_act8_hold(None, 64, 0, 64, 0, 0, None, None, None) == 0  # no rows: nothing to do
    assert L.d3d_act8_restore(16, 1, 10, 64, 0, 5, 1, 64, None) == -1 and b"dtype" in err(L)
    assert L.d3d_act8_restore(16, None, 10, 64, 0, 0, 1, 64, None) == -1 and b"null" in err(L)
    assert L.d3d_act8_restore(16, 1, 10, 64, 0, 0, 1, 60, None) == -1 and b"apart" in err(L)


def test_weight_gradient_refuses(hip_lib):
    L = hip_lib

    def call(fmt=0, n_in=10, cin=64, stride=64, dtype=0, n_out=10, cout=64, nbr=1, cap=10, kvol=27, ws=16, wsb=1 << 40, dy=1):
        return L.d3d_act8_wgrad(16, 1, fmt, n_in, cin, dy, stride, dtype, n_out, cout, nbr, cap, kvol, 1, ws, wsb, None)

    assert call(fmt=3) == -1 and b"format" in err(L)
    assert call(dtype=4) == -1 and b"dtype" in err(L)
    assert call(n_in=0) == -1 and b"n_in" in err(L)
    assert call(n_out=0) == -1
    assert call(cap=9) == -1 and b"cap" in err(L)
    assert call(nbr=None) == -1 and b"kvol" in err(L)
    assert call(nbr=None, kvol=1, n_out=9) == -1
    assert call(kvol=5000) == -1 and b"kvol" in err(L)
    assert call(cin=20000, cout=20000, stride=20000) == -1 and b"weight of" in err(L)
    assert call(stride=63) == -1 and b"apart" in err(L)
    assert call(dy=None) == -1 and b"null" in err(L)
    need = L.d3d_act8_wgrad_workspace_bytes(100000, 27, 64, 64, 0)
    assert need > 0 and call(n_in=100000, n_out=100000, cap=100000, wsb=need - 1) == -2 and b"workspace" in err(L)


def test_row_join_refuses(hip_lib):
    from det3d_amd import _lib

    L = hip_lib

    def fwd(**kw):
        a = dict(n=10, c=64, dtype=0, fmt=0, x=16, x_stride=64, f=16, f_stride=64, pre_kind=1, post_kind=1, h=16, z=16)
        a.update(kw)
        return L.d3d_row_join_fwd(ctypes.byref(_lib.RowJoin(**a)), None)

    for kw, word in ((dict(dtype=2), b"dtype"), (dict(fmt=2), b"format"), (dict(n=0), b"rows"), (dict(c=8193), b"channels"), (dict(x=None), b"no rows"),
                     (dict(x_stride=63), b"x rows"), (dict(f_stride=63), b"f rows"), (dict(x_codes=16), b"codes"), (dict(pre_kind=3), b"kinds"),
                     (dict(pre_eps=-1.0), b"eps"), (dict(pre_eps=float("nan")), b"eps"), (dict(f=None), b"pre norm alone"), (dict(gate=16, gate_cols=5, gate_stride=5), b"gate"),
                     (dict(gate=16, gate_cols=64, gate_stride=5), b"gate"), (dict(gate_act=3), b"gate_act"), (dict(h=None), b"null output"), (dict(z=None), b"null output"),
                     (dict(x_codes=16, x_scales=1), b"together"), (dict(x_codes=8, x_scales=1, f_codes=16, f_scales=1), b"aligned")):
        assert fwd(**kw) == -1 and word in err(L), (kw, err(L))
    assert L.d3d_row_join_fwd(None, None) == -1

    def bwd(a, **kw):
        args = dict(n=10, c=64, dtype=0, fmt=0, x=16, x_stride=64, f=16, f_stride=64, pre_kind=1, post_kind=1)
        args.update(a)
        g = dict(dh=16, dh_stride=64, dz=16, dz_stride=64, dx=16, df=16)
        g.update(kw)
        return L.d3d_row_join_bwd(ctypes.byref(_lib.RowJoin(**args)), ctypes.byref(_lib.RowJoinGrads(**g)), None)

    for a, kw, word in ((dict(), dict(dh_stride=63), b"dh rows"), (dict(), dict(dz_stride=63), b"dz rows"), (dict(pre_kind=0), dict(), b"without a pre"),
                        (dict(f=None, post_kind=0), dict(df=None), b"without f"), (dict(), dict(dgate=16), b"without a gate"),
                        (dict(), dict(dscale=16), b"absent vector"), (dict(x_codes=16, x_scales=1), dict(), b"f is not"),
                        (dict(scale=16, n=100000), dict(dscale=16), None)):
        rc = bwd(a, **kw)
        assert (rc == -1 and word in err(L)) if word else (rc == -2 and b"workspace" in err(L)), (a, kw, err(L))


def test_python_layer_without_a_gpu():
    from det3d_amd import _lib, act8, rownorm

    x = torch.zeros(4, 32)
    with pytest.raises(_lib.D3dError, match="GPU only"):
        act8.hold(x)
    with pytest.raises(ValueError, match="format"):
        act8.hold(x, "int7")
    m = rownorm.RowNorm(32)
    with pytest.raises(_lib.D3dError, match="GPU only"):
        m(x)
    with pytest.raises(_lib.D3dError, match="GPU only"):
        rownorm.join(x, x, pre=m)
    assert m.bias is None and rownorm.RowNorm(32, kind="layer").bias is not None and rownorm.RowNorm(8, affine=False).weight is None
    assert [k for k, _ in rownorm.RowNorm(32, kind="layer").named_parameters()] == ["weight", "bias"]
    for bad in (dict(num_features=0), dict(num_features=8193), dict(num_features=8, kind="group")):
        with pytest.raises(ValueError):
            rownorm.RowNorm(**bad)


def test_buffer_loads_carry_their_whole_offset_where_it_is_checked():
    """The range check of a raw buffer access covers the vector offset; the scalar offset comes on top of it, unchecked.  The weight
    gradient's table entries are requested up to two chunks of rows ahead and rely on the check behind the table's end, so nothing
    that moves may stand in the scalar offset: it is the literal 0."""
    import os
    import re

    from conftest import ROOT

    place = {"load": 2, "store": 3, "load_lds": 4}  # the scalar offset's place among the arguments
    seen = 0
    for name in ("d3d_common.h", "d3d_act8.h", "d3d_act8.hip", "d3d_rownorm.hip"):
        text = open(os.path.join(ROOT, "det3d_amd", "csrc", name)).read()
        for m in re.finditer(r"__builtin_amdgcn_raw_(?:ptr_)?buffer_(load_lds|load|store)\w*\(", text):
            depth, args, at = 1, [""], m.end()
            while depth:
                ch = text[at]
                depth += (ch in "([{") - (ch in ")]}")
                if ch == "," and depth == 1:
                    args.append("")
                elif depth:
                    args[-1] += ch
                at += 1
            seen += 1
            assert args[place[m.group(1)]].strip() == "0", (name, text[m.start():at])
    assert seen >= 5


@pytest.fixture
def launches(hip_lib, monkeypatch):
    """rownorm on CPU tensors with its launches recorded in place of run: (entry point, copies of its description and gradients)"""
    from det3d_amd import act8

    seen = []

    def record(what, dev, fn, *args):
        seen.append((what,) + tuple(type(a._obj).from_buffer_copy(a._obj) for a in args if hasattr(a, "_obj")))

    rows_of = lambda t, what: t if t.stride(1) == 1 and t.stride(0) >= t.shape[1] else t.contiguous()  # noqa: E731
    monkeypatch.setattr(act8, "launch", record)
    monkeypatch.setattr(act8, "rows_of", rows_of)
    return seen


def _join_under_hooks(pack, unpack, checkpoint=None):
    """a join of rows that lie 64 apart, whose saved tensors go through the hooks; (bases, outputs, leaves)"""
    from det3d_amd import rownorm

    bases = [torch.randn(6, 64) for _ in range(3)]
    x, f, gate = (b[:, :32].requires_grad_() for b in bases)
    w = torch.ones(32, requires_grad=True)
    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        ends = rownorm.join(x, f, post=rownorm.NormSpec("rms", w, None, 1e-5), pre=rownorm.NormSpec("rms", None, None, 1e-5), gate=gate, checkpoint=checkpoint)
    return bases, ends, (x, f, gate, w)


def _gradients(ends, leaves):
    return torch.autograd.grad(ends, leaves, (torch.ones(6, 32), torch.ones(6, 32)))


def test_saved_rows_that_come_back_with_other_strides_at_their_address(launches):
    """hooks that pack what is saved give back contiguous copies; where one lies at the address of the strided rows that it was
    taken from, its rows are read at their new distance"""

    def unpack(t):  # (rows: contiguous, at the strided ones' address)
        return t if t.dim() == 1 else torch.as_strided(t.detach(), (6, 32), (32, 1))

    bases, ends, leaves = _join_under_hooks(lambda t: t, unpack)
    _gradients(ends, leaves)
    (_, fwd), (_, bwd, _) = launches
    assert (fwd.x_stride, fwd.f_stride, fwd.gate_stride) == (64, 64, 64)
    assert (bwd.x, bwd.f, bwd.gate) == tuple(b.data_ptr() for b in bases)
    assert (bwd.x_stride, bwd.f_stride, bwd.gate_stride) == (32, 32, 32)


@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_saved_tensors_that_come_back_in_another_layout(launches, checkpoint):
    """columns at a distance, transposed rows, strided vectors and buffers: laid out again before the kernel reads them"""
    kept = []

    def unpack(t):
        wide = torch.zeros(t.shape + (2,), dtype=t.dtype)
        wide[..., 0] = t.detach()
        kept.append(wide)
        return wide[..., 0]

    _, ends, leaves = _join_under_hooks(lambda t: t.clone(), unpack, checkpoint)
    _gradients(ends, leaves)
    bwd = launches[1][1]
    strided = {k.data_ptr() for k in kept}
    rows = (bwd.gate, bwd.post_weight) + ((bwd.x, bwd.f) if checkpoint is None else (bwd.x_codes, bwd.f_codes))
    assert len(kept) == 4 and not strided & set(rows) and bwd.gate_stride == 32
    if checkpoint is None:
        assert (bwd.x_stride, bwd.f_stride) == (32, 32)


def test_saved_tensors_that_come_back_as_something_else(launches):
    from det3d_amd._lib import D3dError

    for unpack in (lambda t: t.bfloat16(), lambda t: t[:1]):
        _, ends, leaves = _join_under_hooks(lambda t: t.clone(), unpack)
        with pytest.raises(D3dError, match="came back"):
            _gradients(ends, leaves)
    assert all(what == "d3d_row_join_fwd" for what, *_ in launches)


def test_forward_mode_derivatives_are_refused(launches):
    """a dual tensor has no requires_grad: without a check its tangent would be dropped, which reads as zero"""
    from torch.autograd import forward_ad

    from det3d_amd import rownorm
    from det3d_amd._lib import D3dError

    x, f, w = torch.randn(3, 8), torch.randn(3, 8), torch.ones(8)
    spec = rownorm.NormSpec("rms", w, None, 1e-5)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, torch.ones_like(x))
        dw = forward_ad.make_dual(w, torch.ones_like(w))
        for bad in (lambda: rownorm.norm(d, spec), lambda: rownorm.norm(x, spec._replace(weight=dw)), lambda: rownorm.join(x, d, post=spec),
                    lambda: rownorm.join(x, f, post=spec, gate=d), lambda: rownorm.join(x, f, pre=spec, scale=dw),
                    lambda: rownorm.norm(d.requires_grad_(), spec)):
            with pytest.raises(D3dError, match="forward-mode"):
                bad()
            with torch.no_grad(), pytest.raises(D3dError, match="forward-mode"):
                bad()
        assert not launches
        rownorm.norm(x, spec)  # plain tensors inside a dual level are nothing special
    rownorm.norm(x, spec)
    assert len(launches) == 2


def test_a_join_without_a_pre_norm_asks_for_no_x(hip_lib):
    """dH = dh there: the backward pass takes f alone, held or not, and the forward pass writes the codes of f alone"""
    from det3d_amd import _lib

    L = hip_lib

    def bwd(**kw):  # (the missing workspace is found behind every other check)
        args = dict(n=100000, c=64, dtype=0, fmt=0, post_kind=1, pre_kind=0, scale=16, f_stride=64)
        args.update(kw)
        rc = L.d3d_row_join_bwd(ctypes.byref(_lib.RowJoin(**args)), ctypes.byref(_lib.RowJoinGrads(dh=16, dh_stride=64, dx=16, df=16, dscale=16)), None)
        return rc, err(L)

    for kw in (dict(f=16), dict(f_codes=16, f_scales=1), dict(f=16, x=16, x_stride=64), dict(f_codes=16, f_scales=1, x_codes=16, x_scales=1)):
        rc, word = bwd(**kw)
        assert rc == -2 and b"workspace" in word, (kw, word)
    for kw, word in ((dict(f=16, pre_kind=1), b"no rows"), (dict(f_codes=16, f_scales=1, pre_kind=1), b"no rows"), (dict(f_codes=16, f_scales=1, x=16, x_stride=64, pre_kind=1), b"together"),
                     (dict(f=16, x_codes=16, x_scales=1), b"f is not")):
        rc, got = bwd(**kw)
        assert rc == -1 and word in got, (kw, got)
    fwd = lambda **kw: L.d3d_row_join_fwd(ctypes.byref(_lib.RowJoin(**{**dict(n=10, c=64, x=16, x_stride=64, f=16, f_stride=64, pre_kind=0), **kw})), None)  # noqa: E731
    assert fwd(f_codes=16, f_scales=1) == -1 and b"null output" in err(L)  # (h is what is missing)
    assert fwd(x_codes=16, x_scales=1) == -1 and b"together" in err(L)
    assert fwd(f_codes=16, f_scales=1, pre_kind=1) == -1 and b"together" in err(L)


@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_a_join_without_a_pre_norm_keeps_no_x(launches, checkpoint):
    """x is neither saved, nor held, nor guarded against a change in place"""
    from det3d_amd import act8, rownorm

    x, f, gate = (torch.randn(6, 40).requires_grad_() for _ in range(3))
    w = torch.ones(40, requires_grad=True)
    stream, kept = x * 1, []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t):
        h = rownorm.join(stream, f, post=rownorm.NormSpec("rms", w, None, 1e-5), gate=gate, checkpoint=checkpoint)
    sizes = [t.numel() * t.element_size() for t in kept]
    assert sorted(sizes) == sorted([6 * 40 * 4, 40 * 4, 6 * 40 * 4 if checkpoint is None else act8.held_bytes(6, 40)])
    with torch.no_grad():
        stream.add_(1)
    dx, *_ = torch.autograd.grad(h, (x, f, gate, w), torch.ones(6, 40))
    assert dx.shape == x.shape
    (_, fwd), (_, bwd, _) = launches
    assert fwd.x == stream.data_ptr() and not fwd.x_codes and bool(fwd.f_codes) == (checkpoint is not None)
    assert not bwd.x and not bwd.x_codes and bool(bwd.f) == (checkpoint is None) and bool(bwd.f_codes) == (checkpoint is not None)


def test_codes_of_an_absent_f_are_refused(hip_lib):
    """a forward pass without f would leave room given for f's codes unwritten"""
    from det3d_amd import _lib

    a = dict(n=10, c=64, x=16, x_stride=64, pre_kind=1, z=16, x_codes=16, x_scales=1, f_codes=16, f_scales=1)
    assert hip_lib.d3d_row_join_fwd(ctypes.byref(_lib.RowJoin(**a)), None) == -1 and b"codes of f without f" in err(hip_lib)


def test_what_the_weight_gradient_can_read(hip_lib):
    """act8.readable is what the entry point accepts, on both sides of every limit"""
    from det3d_amd import act8

    L = hip_lib
    sides = set()
    for n_in, cin, cout, kvol, cap in ((1000, 16, 16, 27, 200000), ((1 << 24) - 1, 16, 16, 27, 200000), (1 << 24, 16, 16, 27, 200000), (1 << 22, 511, 16, 1, 200000),
                                       ((1 << 22) - 1, 512, 16, 1, 200000), (1 << 22, 512, 16, 1, 200000), (1000, 16, 16, 27, (1 << 29) // 27), (1000, 16, 16, 27, (1 << 29) // 27 + 1),
                                       (1000, 16, 16, 1, 1 << 29), (1000, 1, 1, 4096, 100000), (1000, 1, 1, 4097, 100000)):
        # (the missing workspace is found behind every other check)
        rc = L.d3d_act8_wgrad(16, 1, 0, n_in, cin, 1, cout, 0, 100000, cout, 1, cap, kvol, 1, None, 0, None)
        ok = act8.readable(n_in, cin, cout, kvol, cap)
        assert rc == (-2 if ok else -1), (n_in, cin, cout, kvol, cap, rc, err(L))
        sides.add(ok)
    assert sides == {True, False}
    assert not act8.readable(10, 1 << 15, 1 << 15, 1, 10) and L.d3d_act8_wgrad(16, 1, 0, 10, 1 << 15, 1, 1 << 15, 0, 10, 1 << 15, 1, 10, 1, 1, None, 0, None) == -1


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("n,c", [(1, 1), (100, 64), (5000, 24), (2057, 333), (100000, 64), (8192, 4096), (3000, 8192), (1 << 33, 16)])
def test_the_workspace_of_the_column_sums_is_what_they_need(hip_lib, n, c, dtype):
    """one float less is refused: for all five results, and for one alone"""
    from det3d_amd import _lib

    L = hip_lib
    for count, names in ((5, ("dscale", "dpost_weight", "dpost_bias", "dpre_weight", "dpre_bias")), (1, ("dpre_weight",)), (1, ("dpost_bias",))):
        need = L.d3d_row_join_ws_floats(n, c, dtype, count)
        a = _lib.RowJoin(n=n, c=c, dtype=dtype, x=16, x_stride=c, f=16, f_stride=c, scale=16, pre_kind=1, post_kind=1, post_weight=16, post_bias=16, pre_weight=16, pre_bias=16)
        g = _lib.RowJoinGrads(dh=16, dh_stride=c, dz=16, dz_stride=c, ws=16, ws_floats=need - 1, **{k: 16 for k in names})
        assert need > 0 and need % c == 0
        assert L.d3d_row_join_bwd(ctypes.byref(a), ctypes.byref(g), None) == -2 and b"workspace" in err(L), (count, need)
    if (n, c, dtype) == (8192, 4096, 1):
        assert L.d3d_row_join_ws_floats(n, c, dtype, 5) * 4 == 512 * 4 * 4096 * 4  # 34 MB: two blocks of 512 threads a CU


def test_restoring_into_a_tensor_is_a_change_in_place(launches):
    """as with any operation in place: a graph that saved `out` notices, a leaf that wants a gradient is refused"""
    from det3d_amd import act8
    from det3d_amd._lib import D3dError

    held, out, w = act8.hold(torch.randn(4, 32)), torch.ones(4, 32), torch.ones(4, 32, requires_grad=True)
    y = out * w
    assert held.restore(out=out) is out
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with pytest.raises(D3dError, match="requires a gradient"):
        held.restore(out=w)
    with torch.no_grad():
        held.restore(out=w)
    with torch.inference_mode():
        held.restore(out=torch.empty(4, 32))
    assert [what for what, *_ in launches] == ["d3d_act8_hold"] + 3 * ["d3d_act8_restore"]
