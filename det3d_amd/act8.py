"""Activations held in 8 bits between the forward and the backward pass, and the weight gradient that reads them.

A layer keeps its input rows for its weight gradient, a normalisation its input for its own backward pass: most of a training
step's memory.  `hold` keeps such rows `[n, c]` (float32 or bfloat16) as one byte a value: every 32 consecutive channels of a
row share a scale 2^s (one more byte), so a row of whole groups takes 1.03 bytes a value in place of 4 or 2.  Rows are padded to
whole groups: one of 16 channels takes 33 bytes, in place of 64 or 32 (`smaller`).

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


def held_bytes(n, c):
    """size of the buffer that holds n rows of c channels: the codes and one scale a group"""
    p = pitch(c)
    return n * (p + p // GROUP)


def smaller(c, dtype):
    """do rows of c channels take less room in 8 bits?  Not where padding to whole groups eats what the codes save: 16 bfloat16
    channels are 32 bytes a row, held they are 33."""
    return held_bytes(1, c) < c * dtype.itemsize


def readable(n_in, cin, cout, kvol, cap):
    """can `weight_grad` read n_in held rows through a table [kvol, cap]?  (It addresses the table and the codes behind it with 32
    bits: the limits that d3d_act8_wgrad refuses beyond.)"""
    return n_in < 1 << 24 and n_in * pitch(cin) < (1 << 31) - 16 and kvol * cap < 1 << 29 and kvol <= 4096 and kvol * cin * cout < 1 << 30


def rows_of(t, what):
    """`t` as the kernels read a matrix of rows: on the GPU, [n, c], float32 or bfloat16, neighbouring channels next to each
    other (any distance between rows; other layouts are copied)"""
    if not t.is_cuda:
        raise _lib.D3dError("%s runs on the GPU only (HIP kernels); got a %s tensor" % (what, t.device))
    if t.dtype not in _DT:
        raise _lib.D3dError("%s supports float32 / bfloat16 rows, got %s" % (what, t.dtype))
    if t.dim() != 2:
        raise _lib.D3dError("%s: rows [n, c] expected, got shape %s" % (what, tuple(t.shape)))
    n, c = t.shape
    if c < 1:
        raise _lib.D3dError("%s: rows of no channels" % what)
    s0, s1 = t.stride()
    if (s1 != 1 and c > 1) or (s0 < c and n > 1):
        t = t.contiguous()
    return t


def row_stride(t):
    n, c = t.shape
    return t.stride(0) if n > 1 else c


_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device


def launch(what, dev, fn, *args):
    """fn(*args, stream) on the current stream of `dev`, with `dev` as the current device (a launch on a stream of another device
    than the current one is an error of the runtime)"""
    idx = dev.index
    prev = _device()
    if prev != idx:
        torch.cuda.set_device(idx)
    try:
        rc = fn(*args, _lib.stream_ptr(idx))
    finally:
        if prev != idx:
            torch.cuda.set_device(prev)
    if rc:
        _lib.check(rc, what)


class Held:
    """rows held in 8 bits: `shape`, the `dtype` they had, `fmt`, and one buffer with the `codes` (uint8 [n, pitch(c)]) and behind
    them the `scales` (uint8 [n, pitch(c) / 32]: the biased exponent s + 127; 255: a group that is restored as NaN)"""

    __slots__ = ("buf", "shape", "dtype", "fmt", "lease")

    def __init__(self, buf, shape, dtype, fmt, lease):
        self.buf, self.shape, self.dtype, self.fmt, self.lease = buf, shape, dtype, fmt, lease

    @staticmethod
    def room(n, c, dtype, fmt, dev, lease):
        return Held(mem.empty((held_bytes(n, c),), torch.uint8, dev, lease.arena), (n, c), dtype, fmt, lease)

    @property
    def codes(self):
        n, c = self.shape
        return self.buf[:n * pitch(c)].view(n, pitch(c))

    @property
    def scales(self):
        n, c = self.shape
        return self.buf[n * pitch(c):].view(n, pitch(c) // GROUP)

    def pointers(self):
        n, c = self.shape
        p = self.buf.data_ptr()
        return p, p + n * pitch(c)

    def meta(self):
        """what Held(buf, *meta) needs beside the buffer (for autograd nodes, which keep tensors apart)"""
        return self.shape, self.dtype, self.fmt, self.lease

    def check(self, what):
        return self.lease.check(what)

    def nbytes(self):
        return self.buf.numel()

    def restore(self, dtype=None, out=None):
        """the rows again, in `dtype` (default: the one they had) or into `out` [n, c] (any distance between its rows)"""
        n, c = self.shape
        arena = self.check("act8.restore")
        dev = self.buf.device
        if out is None:
            dtype = self.dtype if dtype is None else dtype
            if dtype not in _DT:
                raise _lib.D3dError("act8.restore writes float32 / bfloat16 rows, got %s" % dtype)
            out, stride = mem.empty((n, c), dtype, dev, arena), c
        else:
            if dtype is not None and dtype != out.dtype:
                raise _lib.D3dError("act8.restore: dtype %s, but out is %s" % (dtype, out.dtype))
            if out.dtype not in _DT:
                raise _lib.D3dError("act8.restore writes float32 / bfloat16 rows, got %s" % out.dtype)
            if tuple(out.shape) != (n, c) or out.device != dev or (c > 1 and out.stride(1) != 1) or (n > 1 and out.stride(0) < c):
                raise _lib.D3dError("act8.restore: out must be [%d, %d] on %s with neighbouring channels next to each other and "
                                    "rows that do not overlap" % (n, c, dev))
            if out.requires_grad and torch.is_grad_enabled():
                raise _lib.D3dError("act8.restore: out requires a gradient, which what is written does not carry")
            stride = row_stride(out)
            if not out.is_inference():  # (a graph that saved `out` is to notice)
                torch.autograd.graph.increment_version(out)
        if n:
            codes, scales = self.pointers()
            launch("d3d_act8_restore", dev, _lib.lib().d3d_act8_restore, codes, scales, n, c, FORMATS[self.fmt], _DT[out.dtype],
                   out.data_ptr(), stride)
        return out


def hold(x, fmt="int8"):
    """`x` [n, c] in 8 bits.  Takes values only: nothing of the result carries a gradient."""
    f = format_id(fmt)
    x = rows_of(x, "act8.hold")
    n, c = x.shape
    held = Held.room(n, c, x.dtype, fmt, x.device, mem.Lease())
    if n:
        codes, scales = held.pointers()
        launch("d3d_act8_hold", x.device, _lib.lib().d3d_act8_hold, x.data_ptr(), row_stride(x), n, c, _DT[x.dtype], f, codes, scales)
    return held


def weight_grad(held, dy, nbr=None):
    """The weight gradient of a layer whose input rows are `held` ([n_in, cin]) and whose output gradient is `dy` [n_out, cout]:

        nbr [kvol, cap] int32 (cap >= n_out, as in a Rulebook):  dw[k] = sum_o x[nbr[k][o]]^T dy[o]   -> float32 [kvol, cin, cout]
        nbr None, n_out == n_in (a linear layer, a 1x1 convolution):  dw = x^T dy                     -> float32 [cin, cout]

    Takes values only, as `hold` does.  Entries of the table outside [0, n_in) are absent neighbours and add nothing; behind a table
    there are limits to the held rows and the table's size (`readable`).  Products are exact to float32 (bfloat16 `dy`: as they are;
    float32 `dy`: in three bfloat16 terms, exact from 2^-110 on, smaller values off by at most 2^-134), sums are float32 in a fixed
    order.  A non-finite value in `dy` (float32: also one beyond bfloat16's range, 3.39e38) makes its column of dw non-finite, for
    every offset: rows meet an absent neighbour as a zero."""
    dy = rows_of(dy, "act8.weight_grad")
    n_in, cin = held.shape
    n_out, cout = dy.shape
    dev = dy.device
    if held.buf.device != dev:
        raise _lib.D3dError("act8.weight_grad: rows held on %s, dy on %s" % (held.buf.device, dev))
    if nbr is None:
        kvol, cap = 1, n_out
        if n_out != n_in:
            raise _lib.D3dError("act8.weight_grad: %d held rows, %d rows of dy and no table" % (n_in, n_out))
        dw = torch.empty((cin, cout), dtype=torch.float32, device=dev)
    else:
        if nbr.dtype != torch.int32 or nbr.dim() != 2 or nbr.device != dev or not nbr.is_contiguous():
            raise _lib.D3dError("act8.weight_grad: nbr must be a contiguous int32 [kvol, cap] tensor on %s" % (dev,))
        kvol, cap = nbr.shape
        if kvol < 1 or cap < n_out:
            raise _lib.D3dError("act8.weight_grad: a table of %d x %d entries for %d rows of dy" % (kvol, cap, n_out))
        dw = torch.empty((kvol, cin, cout), dtype=torch.float32, device=dev)
    launch_weight_grad(held, dy, nbr.data_ptr() if nbr is not None else None, cap, kvol, dw)
    return dw


def launch_weight_grad(held, dy, nbr_ptr, cap, kvol, dw):
    """d3d_act8_wgrad on checked operands; `dw` contiguous float32 of kvol * cin * cout values, overwritten"""
    L = _lib.lib()
    n_in, cin = held.shape
    n_out, cout = dy.shape
    arena = held.check("act8.weight_grad")
    if n_out == 0 or n_in == 0 or cout == 0:
        dw.zero_()
        return
    dev, dt = dy.device, _DT[dy.dtype]
    wsb = L.d3d_act8_wgrad_workspace_bytes(n_out, kvol, cin, cout, dt)
    ws = mem.empty((wsb,), torch.uint8, dev, arena) if wsb else None
    codes, scales = held.pointers()
    launch("d3d_act8_wgrad", dev, L.d3d_act8_wgrad, codes, scales, FORMATS[held.fmt], n_in, cin, dy.data_ptr(), row_stride(dy), dt,
           n_out, cout, nbr_ptr, cap, kvol, dw.data_ptr(), ws.data_ptr() if wsb else None, wsb)
