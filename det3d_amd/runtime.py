"""Run-time configuration of the hot path: the switches that change HOW a step is scheduled (and, `activations` alone, what it
computes).

behaviour that changes a result's timing belongs in the configuration, not in
environment variables read at import.  The variables still exist as DEFAULTS (so that `tools/gpu_job.sh env:VAR=..` A/B
runs keep working), but the authoritative state is here and is settable from code:

    from det3d_amd import runtime
    runtime.configure(wgrad_stream="sparse", pair_kernels="off")
    bench line / logs:  runtime.describe()

  wgrad_stream     "all" | "sparse" | "off": weight gradients of the fused backward nodes on a second stream next to the
                   data-gradient chain (sparse_stack / sparse_block / dense_stack; bit-identical results).  "sparse": not in
                   the dense RPN stack, whose two kernels are both MFMA-bound.  Default "all" (D3D_WGRAD_STREAM=0 -> "off").
  wgrad_priority   stream priority of that second stream (0; 1 = lower than the chain)        [D3D_WGRAD_PRIORITY]
  prefetch_priority stream priority of the geometry stream (0; -1 = its small kernels cut in front -- streams of different
                   priorities have hung on MI355X, so every stream is at the default)             [D3D_PREFETCH_PRIORITY]
  pair_kernels     "off" | "measured" | "all": which f32 sparse launches take the pair-compacted kernel (spconv.PAIR_KERNELS)
  stack_executor   "python" | "c": the fused sparse stack's launches call by call from sparse_stack.py, or from one foreign call
                   per direction (csrc/d3d_stack.hip: same entry points, same order, bit-identical).  Default "python": the
                   executor changes neither the step time nor the process's CPU time per step (15.1 vs 15.3 ms, bf16 and
                   f32 alike, profiles/round6_stack_executor.txt) -- it is not the interpreter that bounds the host
                   [D3D_STACK_EXECUTOR]
  activations      "full" | "int8" | "e4m3": what the sparse convolutions, the BatchNorm sweeps behind them and RowNorm keep for the
                   backward pass -- their rows as they are, or in 8 bits (act8.py) where those are smaller.  The one switch here that
                   changes what a step computes: gradients are taken at the restored rows, and so are the signs of the ReLUs that
                   the BatchNorm sweeps have folded in.  In 8 bits the layers run one by one (the fused sparse nodes keep full
                   rows) and TrainStep leaves its step arena aside, so that rows are freed as the forward pass goes on; default
                   "full"                                                                             [D3D_ACTIVATIONS]
  step_arena       TrainStep's default for its step arena (arena.py)
  geometry_ring    slots of GeometryPrefetcher's arena ring (0 = caching allocator)

Changing `wgrad_priority` / `prefetch_priority` after the streams exist has no effect (streams are created once per
device); configure() raises in that case instead of silently doing nothing.
"""
import os

_VALID = {
    "wgrad_stream": ("all", "sparse", "off"),
    "wgrad_after_dgrad": ("off", "dense", "sparse", "all"),
    "pair_kernels": ("off", "measured", "all"),
    "geometry_gate": ("off", "sparse_fwd"),
    "stack_executor": ("c", "python"),
    "activations": ("full", "int8", "e4m3"),
}
_state = {
    "wgrad_stream": "off" if os.environ.get("D3D_WGRAD_STREAM", "1") == "0" else os.environ.get("D3D_WGRAD_STREAM_MODE", "all"),
    "wgrad_after_dgrad": os.environ.get("D3D_WGRAD_AFTER_DGRAD", "off"),
    "wgrad_priority": int(os.environ.get("D3D_WGRAD_PRIORITY", "0")),
    "prefetch_priority": int(os.environ.get("D3D_PREFETCH_PRIORITY", "0")),
    "pair_kernels": os.environ.get("D3D_PAIR_KERNELS", "off"),
    "step_arena": os.environ.get("D3D_STEP_ARENA", "1") != "0",
    "geometry_ring": int(os.environ.get("D3D_GEOMETRY_RING", "3")),
    "geometry_gate": os.environ.get("D3D_GEOMETRY_GATE", "off"),
    "stack_executor": os.environ.get("D3D_STACK_EXECUTOR", "python"),
    "activations": os.environ.get("D3D_ACTIVATIONS", "full"),
}


def get(name):
    return _state[name]


def describe():
    return dict(_state)


def held_format():
    """the 8-bit format that layers keep their rows in between the two passes, None where they keep them as they are"""
    a = _state["activations"]
    return None if a == "full" else a


def wgrad_side(kind):
    """does the backward node of `kind` ("sparse" | "dense") run its weight gradients on the second stream?"""
    m = _state["wgrad_stream"]
    return m == "all" or (m == "sparse" and kind == "sparse")


def wgrad_after_dgrad(kind):
    """does a layer's weight gradient wait for that layer's data gradient to FINISH (instead of starting next to it)?"""
    m = _state["wgrad_after_dgrad"]
    return m == "all" or m == kind


def configure(**kw):
    from . import prefetch, sparse_stack, spconv

    for k, v in kw.items():
        if k not in _state:
            raise KeyError("det3d_amd.runtime: unknown setting %r (have %s)" % (k, sorted(_state)))
        if k in _VALID and v not in _VALID[k]:
            raise ValueError("det3d_amd.runtime: %s = %r, expected one of %s" % (k, v, _VALID[k]))
        if k == "wgrad_priority" and sparse_stack._SIDE and v != _state[k]:
            raise RuntimeError("det3d_amd.runtime: the weight-gradient stream already exists; set wgrad_priority before the first step")
        if k == "prefetch_priority" and prefetch._RESERVED and v != _state[k]:
            raise RuntimeError("det3d_amd.runtime: the geometry stream already exists; set prefetch_priority before it is reserved")
        _state[k] = v
    # the modules' own variables (what the hot loops read) follow
    sparse_stack.WGRAD_STREAM = _state["wgrad_stream"] != "off"
    spconv.PAIR_KERNELS = _state["pair_kernels"]
    return describe()
