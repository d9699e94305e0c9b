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

There is no CPU fallback: without the library and a GPU every call raises.
"""
from __future__ import annotations

import ctypes

import torch

from . import lib as _lib

ACTIVATIONS = {"none": _lib.ACT_NONE, "relu": _lib.ACT_RELU, "silu": _lib.ACT_SILU, "gelu": _lib.ACT_GELU}
_TYPES = {torch.float32: _lib.TYPE_F32, torch.float16: _lib.TYPE_F16, torch.bfloat16: _lib.TYPE_BF16}
_M64 = (1 << 64) - 1
_INT = (1 << 31) - 1


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


def _check(rc):
    if rc < 0:
        raise _lib.FisrError(f"libfisr_hip error {rc}: {_lib.lib().fisr_last_error(None).decode('utf-8', 'replace')}")


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


def _images(x, what, groups):
    if x.dim() != 4:
        raise ValueError(f"{what}: [N, H, W, C] is wanted, got {tuple(x.shape)}")
    if max(x.shape) > _INT or not -1 <= groups <= _INT:
        raise ValueError(f"{what}: {tuple(x.shape)} in {groups} groups: a size is too large")
    if x.dtype not in _TYPES:
        raise ValueError(f"{what}: float32, float16 or bfloat16 is wanted, got {x.dtype}")
    if not x.is_cuda:
        raise _lib.FisrError(f"{what} is on {x.device}: a GPU tensor is wanted (there is no CPU fallback)")


def _like(t, x, what, dtype=None):
    if t.shape != x.shape or t.dtype != x.dtype or t.device != x.device:
        raise ValueError(f"{what}: {tuple(t.shape)} {t.dtype} on {t.device} does not fit {tuple(x.shape)} {x.dtype} on {x.device}")
    return t


def _param(t, x, shape, what):
    if t is None:
        return None
    if t.shape != shape or t.dtype != torch.float32 or t.device != x.device or not t.is_contiguous():
        raise ValueError(f"{what}: a dense float32 tensor {tuple(shape)} on {x.device} is wanted, got {tuple(t.shape)} {t.dtype} on {t.device}")
    return t.data_ptr()


def _act(act):
    try:
        return ACTIVATIONS[act]
    except (KeyError, TypeError):
        raise ValueError(f"act: one of {', '.join(ACTIVATIONS)} is wanted, got {act!r}") from None


def _drop(dropout, x):
    if dropout is None:
        return None
    if dropout.counter is not None and dropout.counter.device != x.device:
        raise ValueError(f"dropout: the counter is on {dropout.counter.device}, the tensor on {x.device}")
    return dropout.desc


def _stream(x):
    return torch._C._cuda_getCurrentRawStream(x.device.index)


def _workspace(L, x, n, h, w, c, groups, backward):
    nbytes = L.fisr_train_groupnorm_workspace_bytes(n, h, w, c, groups, backward)
    return (torch.empty(nbytes, dtype=torch.uint8, device=x.device) if nbytes else None), nbytes


def group_norm(x, groups, gamma=None, beta=None, *, eps=1e-5, act="none", dropout=None, out=None):
    """drop(act((x - mean) * rstd * gamma + beta)) with the mean and rstd = 1 / sqrt(var + eps) of every image's groups of channels.
    Returns (y, stats), stats [2, N, groups] float32: means and rstd, what group_norm_backward takes.  `out` may be x."""
    _images(x, "x", groups)
    n, h, w, c = x.shape
    L = _lib.lib()
    y = torch.empty((n, h, w, c), dtype=x.dtype, device=x.device) if out is None else _like(out, x, "out")
    stats = torch.empty((2, n, groups), dtype=torch.float32, device=x.device) if groups > 0 else None
    ws, nbytes = _workspace(L, x, n, h, w, c, groups, 0)
    _check(L.fisr_train_groupnorm(x.data_ptr(), _pixel_stride(x, "x"), _param(gamma, x, (c,), "gamma"), _param(beta, x, (c,), "beta"),
                                  y.data_ptr(), _pixel_stride(y, "out"), stats.data_ptr() if stats is not None else None, n, h, w, c, groups, eps, _act(act), _drop(dropout, x),
                                  _TYPES[x.dtype], ws.data_ptr() if nbytes else None, nbytes, _stream(x)))
    return y, stats


def group_norm_backward(dy, x, stats, groups, gamma=None, beta=None, *, act="none", dropout=None, dx=None, dgamma=None, dbeta=None,
                        accumulate=False):
    """Gradients of group_norm: (dx, dgamma, dbeta) from dy, the forward pass' x and stats and the same parameters, activation and
    dropout.  dgamma and dbeta (float32 [C]) are made where they are not given; given ones are overwritten or, with `accumulate`, added
    to.  `dx` may be dy."""
    _images(x, "x", groups)
    _like(dy, x, "dy")
    n, h, w, c = x.shape
    L = _lib.lib()
    dx = torch.empty((n, h, w, c), dtype=x.dtype, device=x.device) if dx is None else _like(dx, x, "dx")
    if accumulate and (dgamma is None or dbeta is None):
        raise ValueError("accumulate: dgamma and dbeta have to be given")
    dgamma = torch.empty(c, dtype=torch.float32, device=x.device) if dgamma is None else dgamma
    dbeta = torch.empty(c, dtype=torch.float32, device=x.device) if dbeta is None else dbeta
    ws, nbytes = _workspace(L, x, n, h, w, c, groups, 1)
    _check(L.fisr_train_groupnorm_bwd(x.data_ptr(), _pixel_stride(x, "x"), dy.data_ptr(), _pixel_stride(dy, "dy"), _param(gamma, x, (c,), "gamma"),
                                      _param(beta, x, (c,), "beta"), _param(stats, x, (2, n, groups), "stats"), dx.data_ptr(),
                                      _pixel_stride(dx, "dx"), _param(dgamma, x, (c,), "dgamma"), _param(dbeta, x, (c,), "dbeta"),
                                      1 if accumulate else 0, n, h, w, c, groups, _act(act), _drop(dropout, x), _TYPES[x.dtype],
                                      ws.data_ptr() if nbytes else None, nbytes, _stream(x)))
    return dx, dgamma, dbeta


def dropout(x, drop, residual=None, out=None):
    """drop(x) [+ residual] on a dense tensor of any shape.  `out` may be x or residual."""
    if x.dtype not in _TYPES:
        raise ValueError(f"x: float32, float16 or bfloat16 is wanted, got {x.dtype}")
    if not x.is_cuda:
        raise _lib.FisrError(f"x is on {x.device}: a GPU tensor is wanted (there is no CPU fallback)")
    y = torch.empty_like(x, memory_format=torch.contiguous_format) if out is None else _like(out, x, "out")
    if residual is not None:
        _like(residual, x, "residual")
    if not (x.is_contiguous() and y.is_contiguous() and (residual is None or residual.is_contiguous())):
        raise ValueError("dropout: dense tensors are wanted (the mask goes by an element's place in one)")
    _check(_lib.lib().fisr_train_dropout(x.data_ptr(), residual.data_ptr() if residual is not None else None, y.data_ptr(), x.numel(),
                                         _drop(drop, x), _TYPES[x.dtype], _stream(x)))
    return y


def dropout_backward(dy, drop, out=None):
    """Gradient of dropout with respect to x (that of the residual is dy itself).  `out` may be dy."""
    return dropout(dy, drop, out=out)
