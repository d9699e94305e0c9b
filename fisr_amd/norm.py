"""Group normalisation with an activation, and dropout, on channels-last tensors (`fisr_train_groupnorm*`, `fisr_train_dropout`,
include/fisr.h): the normalisation and regularisation of a residual block beside the convolutions of fisr_amd/train.py.

    y, stats = group_norm(x, groups, gamma, beta, act="silu", dropout=Dropout(0.1, seed, offset))
    dx, dgamma, dbeta = group_norm_backward(dy, x, stats, groups, gamma, beta, act="silu", dropout=Dropout(0.1, seed, offset))
    z = dropout(y, Dropout(0.1, seed, offset + 1), residual=x)
    dy = dropout_backward(dz, Dropout(0.1, seed, offset + 1))

Tensors are [N, H, W, C] on the GPU, float32, float16 or bfloat16; channels are contiguous and pixels lie at one stride (a dense tensor,
or a range of the channels of one).  gamma, beta, statistics and their gradients are float32.  Calls run on torch's current stream of the
tensors' device; workspaces come from torch's allocator, so a call can be captured into a graph.  The dropout mask is a function of
(seed, offset, element): the backward pass is given the same numbers and nothing is stored.

Autograd does not see these calls: what they return has no gradient function even where an input requires a gradient, and a program calls the
backward functions itself (as the tape of fisr_amd/train.py does).  Tensors that a call is given to write count as changed in place: a
graph that kept one of them for its backward pass raises there.

There is no CPU fallback: without the library and a GPU every call raises.
"""
from __future__ import annotations

import functools

import torch

from . import lib as _lib

ACTIVATIONS = {"none": _lib.ACT_NONE, "relu": _lib.ACT_RELU, "silu": _lib.ACT_SILU, "gelu": _lib.ACT_GELU}
_TYPES = {torch.float32: _lib.TYPE_F32, torch.float16: _lib.TYPE_F16, torch.bfloat16: _lib.TYPE_BF16}
_M64 = (1 << 64) - 1
_INT = (1 << 31) - 1
_ENOMEM = -5                                           # FISR_ENOMEM: the workspace is too small


class Dropout:
    """Probability and place in the random sequence of one dropout: `seed` is the generator's key, `offset` the number of the call (a
    program draws another one for every dropout of every step), `counter` an optional int64 tensor of one element on the GPU that is
    added to `offset` when the kernel runs: a captured graph draws a new mask on every replay if the program advances it in between.
    p is taken to a multiple of 1 / 65536; kept values are scaled by the rate that is realised."""
    __slots__ = ("p", "counter", "desc")

    def __init__(self, p, seed, offset=0, counter=None):
        p = float(p)
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"dropout: p = {p} is not in [0, 1]")
        if counter is not None and (counter.dtype != torch.int64 or counter.numel() != 1 or not counter.is_cuda):
            raise ValueError("dropout: the counter is an int64 tensor of one element on the GPU")
        self.p, self.counter = p, counter
        self.desc = _lib.DropoutDesc(p, int(seed) & _M64, int(offset) & _M64, counter.data_ptr() if counter is not None else None)


class _Entries:
    """The library's entry points, found on first use."""

    def __getattr__(self, name):
        if name not in ("gn", "gn_bwd", "drop", "ws_bytes"):
            raise AttributeError(name)
        L = _lib.lib()
        self.gn, self.gn_bwd, self.drop, self.ws_bytes = (L.fisr_train_groupnorm, L.fisr_train_groupnorm_bwd, L.fisr_train_dropout,
                                                          L.fisr_train_groupnorm_workspace_bytes)
        return self.__dict__[name]


_fn = _Entries()


def _pixel_stride(t, what):
    """Elements from pixel to pixel of an [N, H, W, C] tensor whose pixels lie at one stride."""
    n, h, w, c = t.shape
    if t.is_contiguous():
        return c
    sn, sh, sw, sc = t.stride()
    cs = sw if w > 1 else sh if h > 1 else sn if n > 1 else c
    if (c > 1 and sc != 1) or cs < c or (w > 1 and sw != cs) or (h > 1 and sh != w * cs) or (n > 1 and sn != h * w * cs):
        raise ValueError(f"{what}: strides {tuple(t.stride())} of shape {tuple(t.shape)}: channels have to be contiguous and pixels to lie at one stride")
    if cs > _INT:
        raise ValueError(f"{what}: a pixel stride of {cs} elements is too large")
    return cs


def _type(x):
    """The library's number of x's type, and the index of its device."""
    code = _TYPES.get(x.dtype)
    if code is None:
        raise ValueError(f"x: float32, float16 or bfloat16 is wanted, got {x.dtype}")
    if not x.is_cuda:
        raise _lib.FisrError(f"x is on {x.device}: a GPU tensor is wanted (there is no CPU fallback)")
    return code, x.get_device()


def _images(x, groups):
    shape = x.shape
    if len(shape) != 4:
        raise ValueError(f"x: [N, H, W, C] is wanted, got {tuple(shape)}")
    if (x.numel() > _INT and max(shape) > _INT) or not -1 <= groups <= _INT:
        raise ValueError(f"x: {tuple(shape)} in {groups} groups: a size is too large")
    return shape


def _like(t, x, dev, what):
    if t.shape != x.shape or t.dtype != x.dtype or t.get_device() != dev:
        raise ValueError(f"{what}: {tuple(t.shape)} {t.dtype} on {t.device} does not fit {tuple(x.shape)} {x.dtype} on {x.device}")
    return t


def _param(t, dev, shape, what):
    if t is None:
        return None
    if t.shape != shape or t.dtype != torch.float32 or t.get_device() != dev or not t.is_contiguous():
        raise ValueError(f"{what}: a dense float32 tensor {tuple(shape)} on GPU {dev} is wanted, got {tuple(t.shape)} {t.dtype} on {t.device}")
    return t.data_ptr()


def _act(act):
    try:
        return ACTIVATIONS[act]
    except (KeyError, TypeError):
        raise ValueError(f"act: one of {', '.join(ACTIVATIONS)} is wanted, got {act!r}") from None


def _drop(dropout, dev):
    if dropout is None:
        return None
    if dropout.counter is not None and dropout.counter.get_device() != dev:
        raise ValueError(f"dropout: the counter is on {dropout.counter.device}, the tensor on GPU {dev}")
    return dropout.desc


_stream = torch._C._cuda_getCurrentRawStream          # of a device's index: torch.cuda.current_stream(...).cuda_stream without the object


def _apart(out, out_cs, t, t_cs, what):
    """An output may be the tensor itself or lie beside it, in other channels of the same pixels too, but not across it."""
    a, b, size = out.data_ptr(), t.data_ptr(), t.element_size()
    c, pixels = t.shape[-1], t.numel() // t.shape[-1]
    if (a == b and out_cs == t_cs) or a >= b + ((pixels - 1) * t_cs + c) * size or b >= a + ((pixels - 1) * out_cs + c) * size:
        return
    if out_cs != t_cs or not c * size <= (a - b) % (t_cs * size) <= (t_cs - c) * size:
        raise ValueError(f"{what} overlaps an input that it is not")


def _out(x, out, cs, dev, what):
    """The output tensor and its pixel stride."""
    if out is not None:
        return _like(out, x, dev, what), _pixel_stride(out, what)
    if cs == x.shape[3] and x.is_contiguous():
        return torch.empty_like(x), cs
    return x.new_empty(x.shape), x.shape[3]


def _wrote(*given):
    """Counts the caller's tensors among `given` as changed in place."""
    for t in given:
        if t is not None and not t.is_inference():
            torch.autograd.graph.increment_version(t)


@functools.lru_cache(4096)
def _workspace_bytes(n, h, w, c, groups, backward):
    return _fn.ws_bytes(n, h, w, c, groups, backward)


_several = set()          # calls' shapes, strides and alignments that have asked for a workspace: one launch does not hold them


def group_norm(x, groups, gamma=None, beta=None, *, eps=1e-5, act="none", dropout=None, out=None):
    """drop(act((x - mean) * rstd * gamma + beta)) with the mean and rstd = 1 / sqrt(var + eps) of every image's groups of channels.
    Returns (y, stats), stats [2, N, groups] float32: means and rstd, what group_norm_backward takes.  `out` may be x.  var + eps has to
    be at least 2^-126."""
    n, h, w, c = shape = _images(x, groups)
    code, dev = _type(x)
    if out is None and x.is_contiguous():
        y, x_cs, y_cs = torch.empty_like(x), c, c
    else:
        x_cs = _pixel_stride(x, "x")
        y, y_cs = _out(x, out, x_cs, dev, "out")
        if out is not None and x.numel():
            _apart(y, y_cs, x, x_cs, "out")
    stats = x.new_empty((2, n, groups if groups > 0 else 0), dtype=torch.float32)
    call = (x.data_ptr(), x_cs, _param(gamma, dev, (c,), "gamma"), _param(beta, dev, (c,), "beta"), y.data_ptr(), y_cs, stats.data_ptr(), n, h, w, c, groups,
            eps, _act(act), _drop(dropout, dev), code)
    st = _stream(dev)
    key = (shape, groups, code, x_cs, y_cs, (call[0] | call[4]) & 15)
    rc = _ENOMEM if key in _several else _fn.gn(*call, None, 0, st)
    if rc == _ENOMEM:
        if len(_several) >= 4096:
            _several.clear()
        _several.add(key)
        nbytes = _workspace_bytes(n, h, w, c, groups, 0)
        ws = x.new_empty(nbytes, dtype=torch.uint8)
        rc = _fn.gn(*call, ws.data_ptr(), nbytes, st)
    if rc < 0:
        _lib.check(rc)
    if out is not None:
        _wrote(out)
    return y, stats


def group_norm_backward(dy, x, stats, groups, gamma=None, beta=None, *, act="none", dropout=None, dx=None, dgamma=None, dbeta=None,
                        accumulate=False):
    """Gradients of group_norm: (dx, dgamma, dbeta) from dy, the forward pass' x and stats and the same parameters, activation and
    dropout.  dgamma and dbeta (float32 [C]) are made where they are not given; given ones are overwritten or, with `accumulate`, added
    to.  `dx` may be dy, or x."""
    n, h, w, c = _images(x, groups)
    code, dev = _type(x)
    _like(dy, x, dev, "dy")
    x_cs, dy_cs = _pixel_stride(x, "x"), _pixel_stride(dy, "dy")
    given = None if dx is None and dgamma is None and dbeta is None else (dx, dgamma, dbeta)
    dx, dx_cs = _out(x, dx, x_cs, dev, "dx")
    if given and given[0] is not None and x.numel():
        _apart(dx, dx_cs, dy, dy_cs, "dx")
        _apart(dx, dx_cs, x, x_cs, "dx")
    if accumulate and (dgamma is None or dbeta is None):
        raise ValueError("accumulate: dgamma and dbeta have to be given")
    if dgamma is None:
        dgamma = x.new_empty(c, dtype=torch.float32)
    if dbeta is None:
        dbeta = x.new_empty(c, dtype=torch.float32)
    nbytes = _workspace_bytes(n, h, w, c, groups, 1)
    ws = x.new_empty(nbytes, dtype=torch.uint8)
    rc = _fn.gn_bwd(x.data_ptr(), x_cs, dy.data_ptr(), dy_cs, _param(gamma, dev, (c,), "gamma"), _param(beta, dev, (c,), "beta"),
                    _param(stats, dev, (2, n, groups), "stats"), dx.data_ptr(), dx_cs, _param(dgamma, dev, (c,), "dgamma"),
                    _param(dbeta, dev, (c,), "dbeta"), 1 if accumulate else 0, n, h, w, c, groups, _act(act), _drop(dropout, dev), code,
                    ws.data_ptr(), nbytes, _stream(dev))
    if rc < 0:
        _lib.check(rc)
    if given:
        _wrote(*given)
    return dx, dgamma, dbeta


def dropout(x, drop, residual=None, out=None):
    """drop(x) [+ residual] on a dense tensor of any shape.  `out` may be x or residual."""
    code, dev = _type(x)
    y = torch.empty_like(x) if out is None else _like(out, x, dev, "out")
    if not (x.is_contiguous() and (out is None or out.is_contiguous()) and (residual is None or residual.is_contiguous())):
        raise ValueError("dropout: dense tensors are wanted (the mask goes by an element's place in one)")
    res = _like(residual, x, dev, "residual").data_ptr() if residual is not None else None
    if out is not None and x.numel():
        _apart(y.view(-1), x.numel(), x.view(-1), x.numel(), "out")
        if residual is not None:
            _apart(y.view(-1), x.numel(), residual.view(-1), x.numel(), "out")
    rc = _fn.drop(x.data_ptr(), res, y.data_ptr(), x.numel(), _drop(drop, dev), code, _stream(dev))
    if rc < 0:
        _lib.check(rc)
    if out is not None:
        _wrote(out)
    return y


def dropout_backward(dy, drop, out=None):
    """Gradient of dropout with respect to x (that of the residual is dy itself).  `out` may be dy."""
    return dropout(dy, drop, out=out)
