"""Activations held in 8 bits between the forward and the backward pass, and the weight gradient that reads them.

A layer keeps its input rows for its weight gradient, a normalisation its input for its own backward pass: most of a training
step's memory.  `hold` keeps such rows `[n, c]` (float32 or bfloat16) as one byte a value: every 32 consecutive channels of a
row share a scale 2^s (one more byte), so a step holds 1.03 bytes a value in place of 4 or 2.

    int8   s is the smallest with rint(max|x| 2^-s) <= 127, codes are rint(x 2^-s): off by at most 2^(s-1) = max|x| / 127.5
    e4m3   s is the smallest with max|x| 2^-s <= 448, codes are x 2^-s in e4m3: off by at most 2^-4 of the value, or 2^(s-10)

The scale is a power of two, so scaling rounds nothing and a restored value (a code times 2^s, at most 8 significant bits) is
exact in bfloat16: the matrix instructions of `weight_grad` take it as it is.  (s stays within [-120, 121] / [-110, 119], which keeps
every restored value a finite float; values at the upper end are clipped to the largest code.)  A group that holds a NaN or an
infinity is restored as NaN: an overflow is seen in the backward pass, not clipped away.

    held = act8.hold(x, "int8")           # in the forward pass
    dw = act8.weight_grad(held, dy, nbr)  # in the backward pass: dw[k] = sum_o x[nbr[k][o]]^T dy[o]
    x8 = held.restore()

`spconv` layers and the BatchNorm sweeps behind them keep their rows this way under `runtime.configure(activations="int8")`,
`rownorm.norm` / `rownorm.join` under their `checkpoint` argument.
"""
import torch

from . import _lib, arena as mem

GROUP = 32  # channels of a row that share a scale
FORMATS = {"int8": 0, "e4m3": 1}  # D3D_ACT8_INT8, D3D_ACT8_E4M3
_DT = {torch.float32: _lib.D3D_F32, torch.bfloat16: _lib.D3D_BF16}


def format_id(fmt):
    try:
        return FORMATS[fmt]
    except (KeyError, TypeError):
        raise ValueError("act8: format %r, expected one of %s" % (fmt, sorted(FORMATS))) from None


def pitch(c):
    """bytes from one held row to the next: c rounded up to whole groups (the codes behind channel c are zero)"""
    return (c + GROUP - 1) // GROUP * GROUP


def rows_of(t, what):
    """`t` as the kernels read a matrix of rows: on the GPU, [n, c], float32 or bfloat16, neighbouring channels next to each
    other (any distance between rows; other layouts are copied)"""
    if not t.is_cuda:
        raise _lib.D3dError("%s runs on the GPU only (HIP kernels); got a %s tensor" % (what, t.device))
    if t.dim() != 2:
        raise _lib.D3dError("%s: rows [n, c] expected, got shape %s" % (what, tuple(t.shape)))
    if t.dtype not in _DT:
        raise _lib.D3dError("%s supports float32 / bfloat16 rows, got %s" % (what, t.dtype))
    if t.shape[1] < 1:
        raise _lib.D3dError("%s: rows of no channels" % what)
    if (t.stride(1) != 1 and t.shape[1] > 1) or (t.stride(0) < t.shape[1] and t.shape[0] > 1):
        t = t.contiguous()
    return t


def row_stride(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


class on_device:
    """the device of the tensors as the current one for the launches of the block (a launch on a stream of another device
    than the current one is an error of the runtime)"""

    __slots__ = ("idx", "prev")

    def __init__(self, dev):
        self.idx = dev.index

    def __enter__(self):
        self.prev = torch.cuda.current_device()
        if self.prev != self.idx:
            torch.cuda.set_device(self.idx)

    def __exit__(self, *exc):
        if self.prev != self.idx:
            torch.cuda.set_device(self.prev)
        return False


class Held:
    """rows held in 8 bits: `codes` uint8 [n, pitch(c)], `scales` uint8 [n, pitch(c) / 32] (the biased exponent s + 127; 255: a
    group that is restored as NaN), `shape`, the `dtype` they had, and `fmt`"""

    __slots__ = ("codes", "scales", "shape", "dtype", "fmt", "lease")

    def __init__(self, codes, scales, shape, dtype, fmt, lease):
        self.codes, self.scales, self.shape, self.dtype, self.fmt, self.lease = codes, scales, tuple(shape), dtype, fmt, lease

    def meta(self):
        """what Held(codes, scales, *meta) needs beside the two tensors (for autograd nodes, which keep tensors apart)"""
        return self.shape, self.dtype, self.fmt, self.lease

    def check(self, what):
        return self.lease.check(what)

    def nbytes(self):
        return self.codes.numel() + self.scales.numel()

    def restore(self, dtype=None, out=None):
        """the rows again, in `dtype` (default: the one they had) or into `out` [n, c] (any distance between its rows)"""
        n, c = self.shape
        arena = self.check("act8.restore")
        if out is None:
            out = mem.empty((n, c), self.dtype if dtype is None else dtype, self.codes.device, arena)
        elif dtype is not None and dtype != out.dtype:
            raise _lib.D3dError("act8.restore: dtype %s, but out is %s" % (dtype, out.dtype))
        if out.dtype not in _DT:
            raise _lib.D3dError("act8.restore writes float32 / bfloat16 rows, got %s" % out.dtype)
        if tuple(out.shape) != (n, c) or out.device != self.codes.device or (c > 1 and out.stride(1) != 1) or \
                (n > 1 and out.stride(0) < c):
            raise _lib.D3dError("act8.restore: out must be [%d, %d] on %s with neighbouring channels next to each other and rows "
                                "that do not overlap" % (n, c, self.codes.device))
        if n == 0:
            return out
        dev = out.device
        with on_device(dev):
            _lib.check(_lib.lib().d3d_act8_restore(self.codes.data_ptr(), self.scales.data_ptr(), n, c, FORMATS[self.fmt],
                                                   _DT[out.dtype], out.data_ptr(), row_stride(out), _lib.stream_ptr(dev)),
                       "d3d_act8_restore")
        return out


def hold(x, fmt="int8"):
    """`x` [n, c] in 8 bits.  Takes values only: nothing of the result carries a gradient."""
    f = format_id(fmt)
    x = rows_of(x.detach(), "act8.hold")
    n, c = x.shape
    lease = mem.Lease()
    dev, p = x.device, pitch(c)
    codes = mem.empty((n, p), torch.uint8, dev, lease.arena)
    scales = mem.empty((n, p // GROUP), torch.uint8, dev, lease.arena)
    if n:
        with on_device(dev):
            _lib.check(_lib.lib().d3d_act8_hold(x.data_ptr(), row_stride(x), n, c, _DT[x.dtype], f, codes.data_ptr(),
                                                scales.data_ptr(), _lib.stream_ptr(dev)), "d3d_act8_hold")
    return Held(codes, scales, (n, c), x.dtype, fmt, lease)


def weight_grad(held, dy, nbr=None):
    """The weight gradient of a layer whose input rows are `held` ([n_in, cin]) and whose output gradient is `dy` [n_out, cout]:

        nbr [kvol, cap] int32 (cap >= n_out, as in a Rulebook):  dw[k] = sum_o x[nbr[k][o]]^T dy[o]   -> float32 [kvol, cin, cout]
        nbr None, n_out == n_in (a linear layer, a 1x1 convolution):  dw = x^T dy                     -> float32 [cin, cout]

    Entries of the table outside [0, n_in) are absent neighbours and add nothing.  Products are exact to float32 (bfloat16 `dy`: as
    they are; float32 `dy`: in three bfloat16 terms), sums are float32 in a fixed order.  Non-finite values in `dy` make the
    columns that they reach NaN."""
    dy = rows_of(dy, "act8.weight_grad")
    n_in, cin = held.shape
    n_out, cout = dy.shape
    dev = dy.device
    if held.codes.device != dev:
        raise _lib.D3dError("act8.weight_grad: rows held on %s, dy on %s" % (held.codes.device, dev))
    if nbr is None:
        kvol, cap = 1, n_out
        if n_out != n_in:
            raise _lib.D3dError("act8.weight_grad: %d held rows, %d rows of dy and no table" % (n_in, n_out))
    else:
        if nbr.dtype != torch.int32 or nbr.dim() != 2 or nbr.device != dev or not nbr.is_contiguous():
            raise _lib.D3dError("act8.weight_grad: nbr must be a contiguous int32 [kvol, cap] tensor on %s" % (dev,))
        kvol, cap = nbr.shape
        if kvol < 1 or cap < n_out:
            raise _lib.D3dError("act8.weight_grad: a table of %d x %d entries for %d rows of dy" % (kvol, cap, n_out))
    dw = torch.empty((kvol, cin, cout), dtype=torch.float32, device=dev)
    launch_weight_grad(held, dy, nbr.data_ptr() if nbr is not None else None, cap, kvol, dw)
    return dw if nbr is not None else dw[0]


def launch_weight_grad(held, dy, nbr_ptr, cap, kvol, dw):
    """d3d_act8_wgrad on checked operands; `dw` contiguous float32 [kvol, cin, cout], overwritten"""
    L = _lib.lib()
    n_in, cin = held.shape
    n_out, cout = dy.shape
    dev = dy.device
    arena = held.check("act8.weight_grad")
    if n_out == 0 or n_in == 0:
        dw.zero_()
        return
    dt = _DT[dy.dtype]
    wsb = L.d3d_act8_wgrad_workspace_bytes(n_out, kvol, cin, cout, dt)
    ws = mem.empty((wsb,), torch.uint8, dev, arena) if wsb else None
    with on_device(dev):
        _lib.check(L.d3d_act8_wgrad(held.codes.data_ptr(), held.scales.data_ptr(), FORMATS[held.fmt], n_in, cin, dy.data_ptr(),
                                    row_stride(dy), dt, n_out, cout, nbr_ptr, cap, kvol, dw.data_ptr(),
                                    ws.data_ptr() if wsb else None, wsb, _lib.stream_ptr(dev)), "d3d_act8_wgrad")
