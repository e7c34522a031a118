"""Normalisation of rows `[n, c]` over their channels, and the join of a block fused with the norms around it.

    norm   z = w (x - mu) r + b,  r = 1 / sqrt(var + eps)       kind "layer"
           z = w x r + b,         r = 1 / sqrt(mean x^2 + eps)  kind "rms"
    join   h = x + alpha s act(g) post(f),   z = pre(h)

The statistics of a row are its own: unlike BatchNorm nothing couples the sites of a batch or the ranks of a job (no SyncBN
exchange), and a model that answers runs the same formula as one that trains.  `join` is what stands between two blocks of a
residual stream: the norm behind block i (`post`), its gate g and its residual scale s, the addition to the stream, and the norm
in front of block i + 1 (`pre`) -- one pass over x and f that writes h and z.  Every part may be absent: post None: u = f; gate
None: a factor 1; scale None: alpha alone; pre None: only h comes back.

`checkpoint` ("int8" | "e4m3", act8.py) keeps x and f for the backward pass in 8 bits, written in the same pass as h and z; the
gradients are then those at the restored rows: exactly what the backward pass of `join(restored x, restored f, ...)` gives.
x is kept for the pre norm's statistics alone: a join without `pre` keeps f and the gate.

Sums over a row and over the rows (gradients of weights, biases and scales) are float32 in a fixed order: two identical calls
give the same bits.  Both directions can be captured into a graph; as with any autograd node, an eager graph of the same leaves must
not be alive then (a leaf's node belongs to the stream of the first graph that holds it, and the capture would draw that stream in).
`RowNorm` is the module: `norm_cfg = dict(type="RMS" | "LN")` of the backbones and necks builds it
(nn_utils.build_norm_layer), and SparseBasicBlock joins its identity branch through it.
"""
import collections
import ctypes

import torch
from torch import nn
from torch.autograd import forward_ad

from . import _lib, act8, arena as mem, runtime

KINDS = {"rms": 1, "layer": 2}  # D3D_NORM_RMS, D3D_NORM_LAYER
GATE_ACTS = {"none": 0, "sigmoid": 1, "silu": 2}
MAX_CHANNELS = 8192  # a row stays in registers

NormSpec = collections.namedtuple("NormSpec", ("kind", "weight", "bias", "eps"))
NormSpec.__doc__ = "a row norm: kind \"rms\" | \"layer\", float32 weight and bias [c] (either may be None), eps"
_NONE = (0, 0.0, None, None)


def _vector(t, c, dev, what):
    if t is None:
        return None
    if t.dtype != torch.float32 or t.shape != (c,) or t.device != dev:
        raise _lib.D3dError("rownorm: %s must be float32 [%d] on %s, got %s %s on %s" % (what, c, dev, t.dtype, tuple(t.shape), t.device))
    return t if t.is_contiguous() else t.contiguous()


def _spec(norm, c, dev, what):
    """(kind, eps, weight, bias) of a checked NormSpec / RowNorm / None"""
    if norm is None:
        return _NONE
    kind = KINDS.get(norm.kind)
    if kind is None:
        raise ValueError("rownorm: kind %r of the %s norm, expected one of %s" % (norm.kind, what, sorted(KINDS)))
    eps = float(norm.eps)
    if not eps >= 0:
        raise ValueError("rownorm: eps %r of the %s norm" % (norm.eps, what))
    return kind, eps, _vector(norm.weight, c, dev, what + " weight"), _vector(norm.bias, c, dev, what + " bias")


def _dp(t):
    return None if t is None else t.data_ptr()


def _rows(t):
    """address and row stride of checked rows, (None, 0) of none"""
    return (None, 0) if t is None else (t.data_ptr(), act8.row_stride(t))


class _Call:
    """what both directions of a call know beside the tensors"""

    __slots__ = ("n", "c", "dtype", "dt", "dev", "post", "pre", "gate_cols", "act", "alpha", "fmt", "fmt_id", "has_f")

    def desc(self, x, f, gate, scale, post, pre, h, z, hx, hf):
        """the D3dRowJoin of a launch; post, pre: (weight, bias)"""
        xc, xs = hx.pointers() if hx is not None else (None, None)
        fc, fs = hf.pointers() if hf is not None else (None, None)
        return _lib.RowJoin(self.n, self.c, self.dt, self.fmt_id, *_rows(x), *_rows(f), *_rows(gate), self.gate_cols, self.act,
                            _dp(scale), self.alpha, self.post[0], self.post[1], _dp(post[0]), _dp(post[1]),
                            self.pre[0], self.pre[1], _dp(pre[0]), _dp(pre[1]), _dp(h), _dp(z), xc, xs, fc, fs)


def _call(x, f, post, pre, gate, gate_act, alpha, checkpoint):
    call = _Call()
    n, c = x.shape
    dev, dtype = x.device, x.dtype
    if c > MAX_CHANNELS:
        raise _lib.D3dError("rownorm: rows of %d channels, at most %d" % (c, MAX_CHANNELS))
    call.n, call.c, call.dtype, call.dt, call.dev, call.has_f = n, c, dtype, act8._DT[dtype], dev, f is not None
    call.post, call.pre = _spec(post, c, dev, "post"), _spec(pre, c, dev, "pre")
    call.act = GATE_ACTS.get(gate_act)
    if call.act is None:
        raise ValueError("rownorm.join: gate_act %r, expected one of %s" % (gate_act, sorted(GATE_ACTS)))
    call.alpha = float(alpha)
    call.fmt = checkpoint
    call.fmt_id = 0 if checkpoint is None else act8.format_id(checkpoint)
    call.gate_cols = 0
    if f is not None and (f.dtype != dtype or f.device != dev or f.shape != x.shape):
        raise _lib.D3dError("rownorm.join: x %s %s on %s and f %s %s on %s" % (dtype, tuple(x.shape), dev, f.dtype, tuple(f.shape), f.device))
    if gate is not None:
        call.gate_cols = gate.shape[1]
        if gate.dtype != dtype or gate.device != dev or gate.shape[0] != n or (gate.shape[1] != c and gate.shape[1] != 1):
            raise _lib.D3dError("rownorm.join: gate %s %s on %s for rows %s %s on %s: [n, c] or [n, 1] of x's type"
                                % (gate.dtype, tuple(gate.shape), gate.device, dtype, (n, c), dev))
    return call


def _forward(call, x, f, gate, scale, post, pre, arena, hx=None, hf=None):
    """(outputs, the launch's description; None of no rows)"""
    n, c, dev = call.n, call.c, call.dev
    h = mem.empty((n, c), call.dtype, dev, arena) if f is not None else None
    z = mem.empty((n, c), call.dtype, dev, arena) if call.pre[0] else None
    d = None
    if n:
        d = call.desc(x, f, gate, scale, post, pre, h, z, hx, hf)
        act8.launch("d3d_row_join_fwd", dev, _lib.lib().d3d_row_join_fwd, ctypes.byref(d))
    if f is None:
        return z, d
    return (h if z is None else (h, z)), d


def _addresses(tensors):
    return [None if t is None else t.data_ptr() for t in tensors]


def _strides(x, f, gate):
    """distances within the rows that a description holds beside their addresses (x, f: rows or 8-bit buffers)"""
    return [None if t is None else t.stride() for t in (x, f, gate)]


def _gradient(t, dtype, c):
    """(an output's gradient as rows, its address and row stride)"""
    if t is None:
        return None, None, 0
    if t.dtype != dtype:
        t = t.to(dtype)
    if t.is_contiguous():
        return t, t.data_ptr(), c
    t = act8.rows_of(t, "rownorm")
    return t, t.data_ptr(), act8.row_stride(t)


class _JoinFn(torch.autograd.Function):
    """both operators (f None: the norm alone); the weights travel as tensors of their own so that autograd sees them.

    What the backward pass can know in advance is prepared in the forward pass: autograd runs the former on a thread of its own,
    whose first instructions after a wait are several times slower."""

    @staticmethod
    def forward(ctx, call, x, f, gate, scale, post_w, post_b, pre_w, pre_b):
        lease = mem.Lease()
        hx = hf = None
        keep_x = call.pre[0] != 0  # (dH = dh without a pre norm: the backward pass does not read x)
        if call.fmt is not None:
            hx = act8.Held.room(call.n, call.c, call.dtype, call.fmt, call.dev, lease) if keep_x else None
            hf = act8.Held.room(call.n, call.c, call.dtype, call.fmt, call.dev, lease) if f is not None else None
        out, d = _forward(call, x, f, gate, scale, (post_w, post_b), (pre_w, pre_b), lease.arena, hx, hf)
        ctx.set_materialize_grads(False)
        ctx.call, ctx.lease = call, lease
        # (in 8 bits the backward pass reads the codes alone: x and f are free once nobody else holds them)
        if call.fmt is not None:
            x, f = hx.buf if hx is not None else None, hf.buf if hf is not None else None
        elif not keep_x:
            x = None
        saved = (x, f, gate, scale, post_w, post_b, pre_w, pre_b)
        ctx.save_for_backward(*saved)
        _, _, _, _, need_s, need_pw, need_pb, need_qw, need_qb = ctx.needs_input_grad
        ctx.count = need_s + need_pw + need_pb + need_qw + need_qb
        ctx.floats = _lib.lib().d3d_row_join_ws_floats(call.n, call.c, call.dt, ctx.count) if ctx.count and call.n else 0
        if d is not None:
            d.h = d.z = None
            if x is None or hx is not None:
                d.x = None
            if hf is not None:
                d.f = None
        ctx.desc, ctx.at, ctx.strides = d, _addresses(saved), _strides(x, f, gate)
        return out

    @staticmethod
    def backward(ctx, *grads):
        if torch.is_grad_enabled():
            raise _lib.D3dError("rownorm: its gradients have no derivatives of their own (create_graph)")
        call = ctx.call
        n, c, dev, dtype = call.n, call.c, call.dev, call.dtype
        arena = ctx.lease.check("rownorm")
        saved = ctx.saved_tensors
        dh = dz = None
        if call.has_f:
            dh = grads[0]
            if call.pre[0]:
                dz = grads[1]
        else:
            dz = grads[0]
        if dh is None and dz is None:
            return (None,) * 9
        dh, dh_at, dh_stride = _gradient(dh, dtype, c)
        dz, dz_at, dz_stride = _gradient(dz, dtype, c)
        _, need_x, need_f, need_g, need_s, need_pw, need_pb, need_qw, need_qb = ctx.needs_input_grad
        dx = mem.empty((n, c), dtype, dev, arena) if need_x else None
        df = mem.empty((n, c), dtype, dev, arena) if need_f else None
        dgate = mem.empty((n, call.gate_cols), dtype, dev, arena) if need_g else None
        # scale, post weight, post bias, pre weight, pre bias: those that are asked for, each a row of one buffer
        sums = [None] * 5
        if ctx.count:
            buf = torch.empty((ctx.count, c), dtype=torch.float32, device=dev)
            rows = iter(buf.unbind(0))
            sums = [next(rows) if need else None for need in (need_s, need_pw, need_pb, need_qw, need_qb)]
        if n:
            d = ctx.desc
            # saved tensors that hooks had packed come back elsewhere, and strided ones as a rule contiguous: where the allocator
            # reuses the address of freed strided rows, the address alone looks like theirs
            if _addresses(saved) != ctx.at or _strides(*saved[:3]) != ctx.strides:
                saved, d = _elsewhere(call, ctx.lease, saved)
            ws = mem.empty((ctx.floats,), torch.float32, dev, arena) if ctx.count else None
            g = _lib.RowJoinGrads(dh_at, dh_stride, dz_at, dz_stride, _dp(dx), _dp(df), _dp(dgate), *_addresses(sums), _dp(ws), ctx.floats)
            act8.launch("d3d_row_join_bwd", dev, _lib.lib().d3d_row_join_bwd, ctypes.byref(d), ctypes.byref(g))
        elif ctx.count:
            buf.zero_()
        return (None, dx, df, dgate, *sums)


def _elsewhere(call, lease, saved):
    """(the saved tensors as the kernels read them, the backward pass's description with them where they are now)"""
    n, c, dtype, dev = call.n, call.c, call.dtype, call.dev
    rows = ((n, c), dtype) if call.fmt is None else ((act8.held_bytes(n, c),), torch.uint8)
    vector = ((c,), torch.float32)
    as_rows = lambda t: act8.rows_of(t, "rownorm")  # noqa: E731
    plain = as_rows if call.fmt is None else torch.Tensor.contiguous
    back = []
    for t, (shape, kind), lay in zip(saved, (rows, rows, ((n, call.gate_cols), dtype)) + (vector,) * 5, (plain, plain, as_rows) + (torch.Tensor.contiguous,) * 5):
        if t is not None:
            if tuple(t.shape) != shape or t.dtype != kind or t.device != dev:
                raise _lib.D3dError("rownorm: a saved tensor came back as %s %s on %s, it was %s %s on %s" % (t.dtype, tuple(t.shape), t.device, kind, shape, dev))
            t = lay(t)
        back.append(t)
    x, f, gate, scale, post_w, post_b, pre_w, pre_b = back
    hx = hf = None
    if call.fmt is not None:
        hx = act8.Held(x, (n, c), dtype, call.fmt, lease) if x is not None else None
        hf = act8.Held(f, (n, c), dtype, call.fmt, lease) if f is not None else None
        x = f = None
    return back, call.desc(x, f, gate, scale, (post_w, post_b), (pre_w, pre_b), None, None, hx, hf)


def _apply(call, x, f, gate, scale):
    _, _, pw, pb = call.post
    _, _, qw, qb = call.pre
    operands = (x, f, gate, scale, pw, pb, qw, qb)
    if getattr(forward_ad, "_current_level", 0) >= 0:  # (inside a dual level only: asking a tensor takes most of a microsecond)
        for t in operands:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise _lib.D3dError("rownorm: no forward-mode derivatives (an operand is a dual tensor)")
    if torch.is_grad_enabled():
        for t in operands:
            if t is not None and t.requires_grad:
                return _JoinFn.apply(call, x, f, gate, scale, pw, pb, qw, qb)
    return _forward(call, x, f, gate, scale, (pw, pb), (qw, qb), None)[0]


def norm(x, spec, checkpoint=None):
    """z = norm(x): `x` [n, c] float32 or bfloat16, `spec` a NormSpec or a RowNorm; z has x's type."""
    if spec is None:
        raise ValueError("rownorm.norm: no norm given")
    x = act8.rows_of(x, "rownorm.norm")
    return _apply(_call(x, None, None, spec, None, "none", 1.0, checkpoint), x, None, None, None)


def join(x, f, post=None, pre=None, gate=None, gate_act="none", scale=None, alpha=1.0, checkpoint=None):
    """h = x + alpha * scale * act(gate) * post(f), and z = pre(h) when `pre` is given: returns (h, z), or h without `pre`.

    x, f [n, c] of one type (float32 | bfloat16); post, pre: NormSpec, RowNorm or None; gate [n, c] or [n, 1] of x's type with
    gate_act "none" | "sigmoid" | "silu"; scale float32 [c]; alpha a number (no gradient).  z is computed from h before h is
    rounded to its type."""
    x, f = act8.rows_of(x, "rownorm.join"), act8.rows_of(f, "rownorm.join")
    if gate is not None:
        gate = act8.rows_of(gate, "rownorm.join")
    elif gate_act != "none":
        raise ValueError("rownorm.join: gate_act %r without a gate" % (gate_act,))
    call = _call(x, f, post, pre, gate, gate_act, alpha, checkpoint)
    return _apply(call, x, f, gate, _vector(scale, call.c, call.dev, "scale"))


def kept_format(x, c):
    """the `checkpoint` of layers on rows of x's type with c channels, by runtime "activations" ("full" | "int8" | "e4m3"): none where
    8 bits would not make the rows smaller"""
    fmt = runtime.held_format()
    return fmt if fmt is not None and act8.smaller(c, x.dtype) else None


class RowNorm(nn.Module):
    """The norm as a module: rows [n, c] (features of a SparseConvTensor), or [b, c, ...] over its channels (pillars, maps).
    Keeps its input for the backward pass as `kept_format` says."""

    def __init__(self, num_features, eps=1e-5, kind="rms", affine=True, bias=None):
        """bias: None = as the kind has it usually (layer: yes, rms: no)"""
        super().__init__()
        if kind not in KINDS:
            raise ValueError("RowNorm: kind %r, expected one of %s" % (kind, sorted(KINDS)))
        if not 1 <= num_features <= MAX_CHANNELS:
            raise ValueError("RowNorm: %d channels, at most %d" % (num_features, MAX_CHANNELS))
        self.num_features, self.eps, self.kind = int(num_features), float(eps), kind
        bias = kind == "layer" if bias is None else bool(bias)
        self.weight = nn.Parameter(torch.ones(num_features)) if affine else None
        self.bias = nn.Parameter(torch.zeros(num_features)) if affine and bias else None

    @property
    def spec(self):
        return NormSpec(self.kind, self.weight, self.bias, self.eps)

    def extra_repr(self):
        return "%d, eps=%g, kind=%s, affine=%s, bias=%s" % (self.num_features, self.eps, self.kind, self.weight is not None, self.bias is not None)

    def forward(self, x):
        if x.dim() <= 2:
            return norm(x, self.spec, checkpoint=kept_format(x, self.num_features))
        y = x.movedim(1, -1)  # (channels-last memory: a view of rows; other maps are copied into that order)
        z = norm(y.reshape(-1, x.shape[1]), self.spec, checkpoint=kept_format(x, self.num_features))
        return z.view(y.shape).movedim(-1, 1)
