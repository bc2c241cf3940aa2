"""Operators of a policy's head on the library's own kernels (include/factorysim.h, fm_norm.hip / fm_sample.hip /
fm_distill.hip): layer norm, drawing categories from logits, distillation from a teacher's top logits.

GPU tensors are computed on torch's current stream of their device, CPU tensors by the library's CPU backend (as
``FactoryVecEnv(device=-1)``); there is no other path, a missing library raises.  Inputs may have any leading shape and
row stride; one whose last dimension is not adjacent in memory is copied first.  Nothing synchronises and no buffer is
kept between calls, so each call, forward or backward, can be captured into a graph.  Calls can be traced and compiled
(make_fx, torch.compile: each is one operator there) and differentiated by function transforms.  A backward pass that is
captured needs leaves that no live eager graph holds: torch ties a leaf's gradient to the stream of the graph that first
used it.  A row has at most 2^28 elements.
"""
import ctypes as C
import math
import os

import torch
import torch.nn as nn

from . import _lib

__all__ = ["layer_norm", "LayerNorm", "sample_logits", "distill_loss", "MAX_LISTED"]

MAX_LISTED = _lib.FM_DISTILL_MAX_K  # most categories that distill_loss takes for a row

_DTYPES = {torch.float32: _lib.FM_DTYPE_F32, torch.float16: _lib.FM_DTYPE_F16, torch.bfloat16: _lib.FM_DTYPE_BF16}
_INDEX = (torch.int32, torch.int64)


_NODES = os.path.join(os.path.dirname(os.path.abspath(__file__)), "libfactorysim_torch.so")
_loaded = None


def _library():
    """the library, its operators registered with torch (csrc/fm_torch.cpp)"""
    global _loaded
    if _loaded is None:
        L = _lib.load()
        if not hasattr(L, "fm_layer_norm_forward"):
            raise _lib.FactorySimError(f"{_lib.LIB_PATH} has no operators: rebuild it")
        if not os.path.exists(_NODES):
            raise _lib.FactorySimError(f"{_NODES} not built: run `python __graft_entry__.py build`")
        torch.ops.load_library(_NODES)
        names = ("fm_layer_norm_forward", "fm_layer_norm_backward", "fm_layer_norm_workspace", "fm_distill_forward",
                 "fm_distill_backward", "fm_distill_workspace", "fm_sample_logits", "fm_last_error")
        addresses = (C.c_void_p * len(names))(*(C.cast(getattr(L, n), C.c_void_p).value for n in names))
        bind = C.CDLL(_NODES).fm_torch_bind
        bind.argtypes, bind.restype = [C.POINTER(C.c_void_p), C.c_int64], C.c_bool
        if not bind(addresses, len(names)):
            raise _lib.FactorySimError(f"{_NODES} is of another version than {_lib.LIB_PATH}: rebuild both")
        _loaded = L
    return _loaded


@torch.compiler.assume_constant_result
def _ready():
    """the operators are registered: under torch.compile this runs while the call is traced"""
    _library()
    return True


def _call(op, *args):
    try:
        return op(*args)
    except RuntimeError as e:
        if "factorysim error" in str(e):
            raise _lib.FactorySimError(str(e).split("\n")[0]) from None
        raise


def _rows(t):
    """t as [rows, cols] with adjacent columns: a view where there is one"""
    if t.dim() != 2:
        n = t.shape[-1]
        t = t.reshape(-1 if n else 0, n)
    return t if t.shape[1] <= 1 or t.stride(1) == 1 else t.contiguous()


def _float_input(name, t):
    if not torch.is_tensor(t):
        raise TypeError(f"{name} is a tensor")
    if t.dtype not in _DTYPES:
        raise TypeError(f"{name} is float32, float16 or bfloat16, not {t.dtype}")
    if t.dim() < 1 or t.shape[-1] < 1:
        raise ValueError(f"{name} needs a last dimension of at least 1, got shape {tuple(t.shape)}")
    if not t.is_cuda and t.device.type != "cpu":
        raise ValueError(f"{name} is on {t.device}: a GPU or the CPU is needed")


def _same_device(t, **others):
    for name, o in others.items():
        if o is not None and o.device != t.device:
            raise ValueError(f"{name} is on {o.device}, the first input on {t.device}")


# ------------------------------------------------------------------ layer norm
def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(variance + eps) * weight + bias over the last dimension (biased variance), in x's dtype.

    x: float32, float16 or bfloat16; weight, bias: [x.shape[-1]], both of x's dtype or both float32, or None.  Statistics
    and sums are held in 32 bits and each result is rounded once.  Differentiable once in x, weight and bias; the
    parameters' gradients are summed over rows in a fixed order."""
    _float_input("x", x)
    v = x.shape[-1]
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        if not torch.is_tensor(p):
            raise TypeError(f"{name} is a tensor or None")
        if p.dtype != x.dtype and p.dtype != torch.float32:
            raise TypeError(f"{name} is float32 or of x's dtype {x.dtype}, not {p.dtype}")
        if tuple(p.shape) != (v,):
            raise ValueError(f"{name} has shape {tuple(p.shape)}, x's last dimension is {v}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"weight is {weight.dtype}, bias {bias.dtype}: one dtype for both")
    _same_device(x, weight=weight, bias=bias)
    eps = float(eps)
    if not 0 <= eps < math.inf:
        raise ValueError(f"eps is finite and not negative, got {eps}")
    w = weight if weight is None or weight.is_contiguous() else weight.contiguous()
    b = bias if bias is None or bias.is_contiguous() else bias.contiguous()
    _ready()
    y = _call(torch.ops.factorysim.layer_norm, _rows(x), w, b, eps)
    return y if x.dim() == 2 else y.view(x.shape)


class LayerNorm(nn.Module):
    """``layer_norm`` over the last dimension with a weight (ones at first) and a bias (zeros)"""

    def __init__(self, dim, eps=1e-5):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(dim))
        self.bias = nn.Parameter(torch.zeros(dim))

    def forward(self, x):
        return layer_norm(x, self.weight, self.bias, self.eps)

    def extra_repr(self):
        return f"{self.weight.numel()}, eps={self.eps}"


# ------------------------------------------------------------------ drawing categories
def _row_setting(name, value, rows, logits, dtype):
    """a setting of each row as a contiguous tensor of the library's type"""
    if value.dtype.is_floating_point != (dtype == torch.float32) or value.dtype in (torch.bool, torch.float64):
        raise TypeError(f"{name} of each row is {'a float32' if dtype == torch.float32 else 'an integer'} tensor, "
                        f"not {value.dtype}")
    if value.numel() != rows or (value.dim() > 1 and value.shape != logits.shape[:-1]):
        raise ValueError(f"{name} has shape {tuple(value.shape)}, the logits' rows {tuple(logits.shape[:-1])}")
    if value.device != logits.device:
        raise ValueError(f"{name} is on {value.device}, the logits on {logits.device}")
    if value.dtype == torch.int64:  # beyond any number of categories is off, as 0 is
        value = value.clamp(0, 2**31 - 1)
    return value.reshape(-1).to(dtype).contiguous()


def sample_logits(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, mask=None):
    """One category of each row of ``logits`` [..., categories], drawn with the uniform numbers ``u`` [...]: int64 [...].

    A row's categories are ranked by logit, the lower index first among equals, and weigh exp(logit / temperature).
    ``top_k`` keeps the first k, ``top_p`` the shortest leading part of those that holds at least that share of their
    weight, ``min_p`` those of them that weigh at least that share of the largest.  The result is the first of the kept
    categories, in rank, up to which more than the share u of their weight lies: u = 0 gives the largest logit.

    Each setting is a number or a tensor with one number for each row (float32; ``top_k`` integer).  temperature <= 0
    gives the largest logit; top_k <= 0, top_p >= 1 and min_p <= 0 are off.  ``mask`` (bool, logits' shape or
    [categories]) bars categories where it is False, whatever their logit; a logit of -inf bars its category too.
    -1 stands for a row with no category left, with NaN in a logit that is not barred, or with a NaN in u or a setting.
    logits: float32, float16 or bfloat16; u: float32 or float64, in [0, 1).  Weights below 2^-52 of the largest count as
    nothing, on the GPU beyond 2048 categories those below e^-33 (2^-47.6), beyond 2^15 below 2^-47, twice that for each doubling.
    The same call draws the same on every run; where a border falls within 5e-13 of the row's weight of one between two
    categories, the GPU and the CPU may draw neighbours."""
    _float_input("logits", logits)
    if not torch.is_tensor(u) or u.dtype not in (torch.float32, torch.float64):
        raise TypeError("u is a float32 or float64 tensor")
    if u.shape != logits.shape[:-1]:
        raise ValueError(f"u has shape {tuple(u.shape)}, the logits' rows {tuple(logits.shape[:-1])}")
    if u.device != logits.device:
        raise ValueError(f"u is on {u.device}, the logits on {logits.device}")
    z = _rows(logits)
    n, v = z.shape
    m = None
    if mask is not None:
        if not torch.is_tensor(mask) or mask.dtype != torch.bool:
            raise TypeError(f"mask is a bool tensor, not {getattr(mask, 'dtype', type(mask))}")
        if mask.shape != logits.shape and tuple(mask.shape) != (v,):
            raise ValueError(f"mask has shape {tuple(mask.shape)}, the logits {tuple(logits.shape)}")
        if mask.device != logits.device:
            raise ValueError(f"mask is on {mask.device}, the logits on {logits.device}")
        m = _rows(mask if mask.shape == logits.shape else mask[None])
    t_rows = k_rows = p_rows = q_rows = None
    if torch.is_tensor(temperature):
        temperature, t_rows = 0.0, _row_setting("temperature", temperature, n, logits, torch.float32)
    if torch.is_tensor(top_k):
        top_k, k_rows = 0, _row_setting("top_k", top_k, n, logits, torch.int32)
    if torch.is_tensor(top_p):
        top_p, p_rows = 0.0, _row_setting("top_p", top_p, n, logits, torch.float32)
    if torch.is_tensor(min_p):
        min_p, q_rows = 0.0, _row_setting("min_p", min_p, n, logits, torch.float32)
    t, p, q, k = float(temperature), float(top_p), float(min_p), int(top_k)
    if t != t or p != p or q != q:
        raise ValueError("temperature, top_p and min_p are numbers, not NaN")
    u = u.reshape(-1).contiguous() if u.dim() != 1 or not u.is_contiguous() else u
    _ready()
    out = _call(torch.ops.factorysim.sample_logits, z, u, m, t, min(max(k, 0), 2**31 - 1), p, q, t_rows, k_rows, p_rows, q_rows)
    return out if logits.dim() == 2 else out.view(logits.shape[:-1])


# ------------------------------------------------------------------ distillation
def distill_loss(logits, teacher_index, teacher_logits, temperature=1.0):
    """temperature^2 times the Kullback-Leibler divergence of softmax(logits / temperature) over all categories from
    softmax(teacher_logits / temperature) over the listed ones, for each row: float32 [...].

    logits [..., categories] (float32, float16 or bfloat16); teacher_index [..., k] (int32 or int64) names the listed
    categories and teacher_logits [..., k] (a float dtype of its own) their logits, k at most 1024, in any order.  An
    entry with a negative index or a teacher logit of -inf is not listed (lists of unequal length are padded so); a row
    with none has loss 0 and gradient 0.  A category listed twice counts twice.  An index that is no category cannot be raised
    without waiting for the GPU: it makes its row's loss and gradient NaN, as do logits without a softmax (all -inf, or
    NaN or +inf among them or the listed teacher's).  Differentiable once in the logits; the
    teacher's logits are constants."""
    _float_input("logits", logits)
    _float_input("teacher_logits", teacher_logits)
    if not torch.is_tensor(teacher_index) or teacher_index.dtype not in _INDEX:
        raise TypeError("teacher_index is an int32 or int64 tensor")
    if teacher_index.shape != teacher_logits.shape or teacher_index.shape[:-1] != logits.shape[:-1]:
        raise ValueError(f"teacher_index {tuple(teacher_index.shape)} and teacher_logits {tuple(teacher_logits.shape)} "
                         f"list categories for each row of the logits {tuple(logits.shape)}")
    if teacher_index.shape[-1] > MAX_LISTED:
        raise ValueError(f"at most {MAX_LISTED} categories can be listed, got {teacher_index.shape[-1]}")
    if teacher_logits.requires_grad:
        raise ValueError("teacher_logits requires a gradient, which this loss does not give: detach it")
    _same_device(logits, teacher_index=teacher_index, teacher_logits=teacher_logits)
    temperature = float(temperature)
    if not 1e-30 <= temperature <= 1e30:
        raise ValueError(f"temperature is positive and within 1e-30 .. 1e30, got {temperature}")
    _ready()
    loss = _call(torch.ops.factorysim.distill_loss, _rows(logits), _rows(teacher_index), _rows(teacher_logits), temperature)
    return loss if logits.dim() == 2 else loss.view(logits.shape[:-1])
