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

Sums over a row and over the rows (gradients of weights, biases and scales) are float32 in a fixed order: two identical calls
give the same bits.  `RowNorm` is the module: `norm_cfg = dict(type="RMS" | "LN")` of the backbones and necks builds it
(nn_utils.build_norm_layer), and SparseBasicBlock joins its identity branch through it.
"""
import collections
import ctypes

import torch
from torch import nn

from . import _lib, act8, arena as mem, runtime

KINDS = {"rms": 1, "layer": 2}  # D3D_NORM_RMS, D3D_NORM_LAYER
GATE_ACTS = {"none": 0, "sigmoid": 1, "silu": 2}
MAX_CHANNELS = 8192  # a row stays in registers

NormSpec = collections.namedtuple("NormSpec", ("kind", "weight", "bias", "eps"))
NormSpec.__doc__ = "a row norm: kind \"rms\" | \"layer\", float32 weight and bias [c] (either may be None), eps"
_NONE = NormSpec(None, None, None, 0.0)


def _vector(t, c, dev, what):
    if t is None:
        return None
    if t.dtype != torch.float32 or t.dim() != 1 or t.shape[0] != c or t.device != dev:
        raise _lib.D3dError("rownorm: %s must be float32 [%d] on %s, got %s %s on %s" % (what, c, dev, t.dtype, tuple(t.shape), t.device))
    return t if t.is_contiguous() else t.contiguous()


def _spec(norm, c, dev, what):
    if norm is None:
        return _NONE
    if isinstance(norm, RowNorm):
        norm = norm.spec
    if norm.kind not in KINDS:
        raise ValueError("rownorm: kind %r of the %s norm, expected one of %s" % (norm.kind, what, sorted(KINDS)))
    if not norm.eps >= 0:
        raise ValueError("rownorm: eps %r of the %s norm" % (norm.eps, what))
    return NormSpec(norm.kind, _vector(norm.weight, c, dev, what + " weight"), _vector(norm.bias, c, dev, what + " bias"), float(norm.eps))


class _Call:
    """one call's operands, checked: what fills the D3dRowJoin of both directions"""

    __slots__ = ("n", "c", "dtype", "dev", "post", "pre", "gate_cols", "act", "alpha", "fmt")

    def __init__(self, x, f, post, pre, gate, gate_act, scale, alpha, checkpoint):
        n, c = x.shape
        if c > MAX_CHANNELS:
            raise _lib.D3dError("rownorm: rows of %d channels, at most %d" % (c, MAX_CHANNELS))
        self.n, self.c, self.dtype, self.dev = n, c, act8._DT[x.dtype], x.device
        self.post, self.pre = _spec(post, c, x.device, "post"), _spec(pre, c, x.device, "pre")
        if gate_act not in GATE_ACTS:
            raise ValueError("rownorm.join: gate_act %r, expected one of %s" % (gate_act, sorted(GATE_ACTS)))
        self.act, self.alpha = GATE_ACTS[gate_act], float(alpha)
        self.fmt = None if checkpoint is None else checkpoint
        if checkpoint is not None:
            act8.format_id(checkpoint)
        for t, what in ((f, "f"), (gate, "gate")):
            if t is not None and (t.dtype != x.dtype or t.device != x.device):
                raise _lib.D3dError("rownorm.join: %s is %s on %s, x %s on %s" % (what, t.dtype, t.device, x.dtype, x.device))
        if f is not None and f.shape != x.shape:
            raise _lib.D3dError("rownorm.join: x %s and f %s" % (tuple(x.shape), tuple(f.shape)))
        self.gate_cols = 0
        if gate is not None:
            if gate.shape[0] != n or gate.shape[1] not in (1, c):
                raise _lib.D3dError("rownorm.join: gate %s for rows %s: [n, c] or [n, 1]" % (tuple(gate.shape), (n, c)))
            # (c == 1: one value a row either way)
            self.gate_cols = gate.shape[1]

    def desc(self, x, f, gate, scale, h, z, held=(None, None)):
        hx, hf = held
        p, q = self.post, self.pre
        return _lib.RowJoin(
            self.n, self.c, self.dtype, act8.FORMATS[self.fmt] if self.fmt else 0,
            _dp(x), act8.row_stride(x) if x is not None else 0, _dp(f), act8.row_stride(f) if f is not None else 0,
            _dp(gate), act8.row_stride(gate) if gate is not None else 0, self.gate_cols, self.act, _dp(scale), self.alpha,
            KINDS.get(p.kind, 0), p.eps, _dp(p.weight), _dp(p.bias), KINDS.get(q.kind, 0), q.eps, _dp(q.weight), _dp(q.bias),
            _dp(h), _dp(z),
            hx.codes.data_ptr() if hx else None, hx.scales.data_ptr() if hx else None,
            hf.codes.data_ptr() if hf else None, hf.scales.data_ptr() if hf else None)


def _dp(t):
    return None if t is None else t.data_ptr()


def _forward(call, x, f, gate, scale, arena, held=(None, None)):
    n, c, dev = call.n, call.c, call.dev
    h = mem.empty((n, c), x.dtype, dev, arena) if f is not None else None
    z = mem.empty((n, c), x.dtype, dev, arena) if call.pre.kind else None
    if n:
        d = call.desc(x, f, gate, scale, h, z, held)
        with act8.on_device(dev):
            _lib.check(_lib.lib().d3d_row_join_fwd(ctypes.byref(d), _lib.stream_ptr(dev)), "d3d_row_join_fwd")
    return h, z


class _JoinFn(torch.autograd.Function):
    """both operators (f None: the norm alone); the weights travel as tensors of their own so that autograd sees them"""

    @staticmethod
    def forward(ctx, x, f, gate, scale, post_w, post_b, pre_w, pre_b, call):
        lease = mem.Lease()
        hx = hf = None
        if call.fmt:
            n, c, p = call.n, call.c, act8.pitch(call.c)

            def room():
                return act8.Held(mem.empty((n, p), torch.uint8, call.dev, lease.arena),
                                 mem.empty((n, p // act8.GROUP), torch.uint8, call.dev, lease.arena), (n, c), x.dtype, call.fmt, lease)
            hx, hf = room(), room() if f is not None else None
        h, z = _forward(call, x, f, gate, scale, lease.arena, (hx, hf))
        ctx.set_materialize_grads(False)
        ctx.call, ctx.lease, ctx.row_dtype, ctx.has_f = call, lease, x.dtype, f is not None
        # (in 8 bits the backward pass reads the codes alone: x and f are free once nobody else holds them)
        held = () if hx is None else (hx.codes, hx.scales) + ((hf.codes, hf.scales) if hf is not None else ())
        ctx.save_for_backward(*(held or (x, f)), gate, scale, post_w, post_b, pre_w, pre_b)
        if f is None:
            return z
        return h if z is None else (h, z)

    @staticmethod
    def backward(ctx, *grads):
        if torch.is_grad_enabled():
            raise _lib.D3dError("rownorm: its gradients have no derivatives of their own (create_graph)")
        call, has_f = ctx.call, ctx.has_f
        n, c, dev, dtype = call.n, call.c, call.dev, ctx.row_dtype
        saved = ctx.saved_tensors
        gate, scale, post_w, post_b, pre_w, pre_b = saved[-6:]
        x = f = hx = hf = None
        if call.fmt:
            hx = act8.Held(saved[0], saved[1], (n, c), dtype, call.fmt, ctx.lease)
            hf = act8.Held(saved[2], saved[3], (n, c), dtype, call.fmt, ctx.lease) if has_f else None
        else:
            x, f = saved[:2]
        dh, dz = (grads[0] if has_f else None), (grads[-1] if call.pre.kind else None)
        arena = ctx.lease.check("rownorm")
        need = ctx.needs_input_grad
        if dh is None and dz is None:
            return (None,) * 9
        dh, dz = (None if g is None else act8.rows_of(g if g.dtype == dtype else g.to(dtype), "rownorm") for g in (dh, dz))

        def rows(wanted, cols=c):
            return mem.empty((n, cols), dtype, dev, arena) if wanted else None

        dx, df, dgate = rows(need[0]), rows(has_f and need[1]), rows(gate is not None and need[2], call.gate_cols)
        # scale, post weight, post bias, pre weight, pre bias: those that are asked for, each a row of one buffer
        there = (scale, post_w, post_b, pre_w, pre_b)
        want = [t is not None and need[3 + i] for i, t in enumerate(there)]
        sums = list(torch.empty((sum(want), c), dtype=torch.float32, device=dev).unbind(0)) if any(want) else []
        if n:
            L = _lib.lib()
            ws = None
            floats = 0
            if sums:
                floats = L.d3d_row_join_ws_floats(n, c, call.dtype, len(sums))
                ws = mem.empty((floats,), torch.float32, dev, arena) if floats else None
            d = call.desc(x, f, gate, scale, None, None, (hx, hf))
            it = iter(sums)
            ptrs = [next(it).data_ptr() if w else None for w in want]
            g = _lib.RowJoinGrads(_dp(dh), act8.row_stride(dh) if dh is not None else 0, _dp(dz),
                                  act8.row_stride(dz) if dz is not None else 0, _dp(dx), _dp(df), _dp(dgate), *ptrs, _dp(ws), floats)
            with act8.on_device(dev):
                _lib.check(L.d3d_row_join_bwd(ctypes.byref(d), ctypes.byref(g), _lib.stream_ptr(dev)), "d3d_row_join_bwd")
        else:
            for t in sums:
                t.zero_()
        it = iter(sums)
        return (dx, df, dgate) + tuple(next(it) if w else None for w in want) + (None,)


def _apply(x, f, gate, scale, call):
    p, q = call.post, call.pre
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, f, gate, scale, p.weight, p.bias, q.weight, q.bias)):
        return _JoinFn.apply(x, f, gate, scale, p.weight, p.bias, q.weight, q.bias, call)
    h, z = _forward(call, x, f, gate, scale, None)
    if f is None:
        return z
    return h if z is None else (h, z)


def norm(x, spec, checkpoint=None):
    """z = norm(x): `x` [n, c] float32 or bfloat16, `spec` a NormSpec or a RowNorm; z has x's type."""
    if spec is None:
        raise ValueError("rownorm.norm: no norm given")
    x = act8.rows_of(x, "rownorm.norm")
    return _apply(x, None, None, None, _Call(x, None, None, spec, None, "none", None, 1.0, checkpoint))


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
    call = _Call(x, f, post, pre, gate, gate_act, scale, alpha, checkpoint)
    return _apply(x, f, gate, _vector(scale, x.shape[1], x.device, "scale"), call)


class RowNorm(nn.Module):
    """The norm as a module: rows [n, c] (features of a SparseConvTensor), or [b, c, ...] over its channels (pillars, maps).
    Keeps its input for the backward pass as runtime "activations" says ("full" | "int8" | "e4m3")."""

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
            return norm(x, self.spec, checkpoint=runtime.held_format())
        y = x.movedim(1, -1)  # (channels-last memory: a view of rows; other maps are copied into that order)
        z = norm(y.reshape(-1, x.shape[1]), self.spec, checkpoint=runtime.held_format())
        return z.view(y.shape).movedim(-1, 1)
