"""Regularisation of the Q networks' hidden layers: dropout whose mask comes from the counter-based generator and is never stored, group norm
with an activation over channels-last data, and the two in one pass (linear -> dropout -> norm -> activation), each with its gradient.  HIP kernels of
csrc/regularise.hip and regularise_norm.hip behind the C ABI include/plenreg.h, with their autograd nodes in csrc/regularise_torch.cpp;
td3.RegularisedCritic is the framework's own caller.

The twin critics' hidden rows lie side by side in one [B, 512] matrix, so group norm with two groups is both networks' layer norm in one call.

Random state: an int64[2] device tensor {seed, calls so far}, the form every draw of this package uses (`new_rng`).  Which mask a call draws depends
on that state, on `site` (one number per place in the model) and on the element's index alone, not on type, strides or launch shape.  A call only READS the
state; `advance` moves it on, once per iteration, as a kernel (so a captured graph draws new masks at every replay).  The backward pass draws the
forward's mask again from a 16-byte snapshot that the forward kernel takes.  (Who runs a forward pass a second time, as activation checkpointing does, has to do so before
`advance`: it draws from the state as it then stands.)

The kernels are no library operations: a call that is being traced (torch.jit.trace, make_fx, fake tensors) or transformed (vmap, torch.func.grad) is refused.  Under
torch.compile the operators run as they are, between the compiled parts.

CPU tensors take the same definitions as elementary torch operations (autograd differentiates them): the multi-process CPU path of td3.py."""
import ctypes as C
import importlib.util
import math
import os

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.environ.get("PLENREG_LIB") or os.path.join(_HERE, "csrc", "libplenreg.so")
EXPORTS = ["plenreg_dropout", "plenreg_norm_forward", "plenreg_norm_backward", "plenreg_norm_workspace", "plenreg_version"]
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ACTS = {"none": 0, "relu": 1, "silu": 2}
MAX_C, MAX_C_LONG = 32768, 8192           # PLENREG_MAX_C, PLENREG_MAX_C_LONG
MAX_DRAWN = 1 << 35                       # the mask counts blocks of 8 elements in 32 bits
_lib = _nodes = None


class PlenRegError(RuntimeError):
    pass


class DropoutArgs(C.Structure):
    """Mirror of PlenRegDropout (include/plenreg.h), for callers of the C entry points (the operators below go through csrc/regularise_torch.cpp)."""
    _fields_ = ([(n, C.c_void_p) for n in ("x", "y", "rng", "used")] + [(n, C.c_int64) for n in ("rows", "cols", "x_stride")]
                + [("dtype", C.c_int32), ("cut", C.c_uint32), ("site", C.c_int32)])


class NormArgs(C.Structure):
    """Mirror of PlenRegNorm (include/plenreg.h)."""
    _fields_ = ([(n, C.c_void_p) for n in ("x", "dy", "w", "b", "out", "stats", "dw", "db", "ws", "rng", "used")]
                + [(n, C.c_int64) for n in ("N", "L", "x_stride", "dy_stride")] + [(n, C.c_int32) for n in ("C", "G", "dtype", "w_dtype", "act")]
                + [("cut", C.c_uint32), ("site", C.c_int32), ("eps", C.c_float)])


def load():
    """dlopen the HIP library; raises if it has not been built (device tensors have no other path)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise PlenRegError("%s is missing: run `python -c 'import __graft_entry__ as g; g.build()'` (hipcc --offload-arch=gfx950)" % LIB_PATH)
        lib = C.CDLL(LIB_PATH)
        for name in EXPORTS:
            getattr(lib, name)
        lib.plenreg_version.restype = C.c_char_p
        lib.plenreg_dropout.argtypes = [C.POINTER(DropoutArgs), C.c_void_p]
        lib.plenreg_norm_forward.argtypes = lib.plenreg_norm_backward.argtypes = [C.POINTER(NormArgs), C.c_void_p]
        lib.plenreg_norm_workspace.argtypes = [C.POINTER(NormArgs), C.c_int]
        lib.plenreg_norm_workspace.restype = C.c_int64
        _lib = lib
    return _lib


def _load_nodes():
    """The autograd nodes (csrc/regularise_torch.cpp), bound to the HIP library's entry points."""
    global _nodes, _quick_dropout, _quick_norm, _quick_layer
    lib = load()
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "csrc", "plenreg_torch.so")
    if not os.path.exists(path):
        raise PlenRegError("%s is missing: run `python -c 'import __graft_entry__ as g; g.build()'`" % path)
    spec = importlib.util.spec_from_file_location("plenreg_torch", path)
    nodes = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(nodes)
    nodes.bind(*(C.cast(f, C.c_void_p).value for f in (lib.plenreg_dropout, lib.plenreg_norm_forward, lib.plenreg_norm_backward, lib.plenreg_norm_workspace)))
    _nodes = nodes
    _quick_dropout, _quick_norm, _quick_layer = nodes.quick_dropout, nodes.quick_norm, nodes.quick_layer
    return nodes


def _not_loaded(*args):
    return None


# natively: a call whose arguments pass every check below is launched at once; None where one does not, or before the first call on a device
_quick_dropout = _quick_norm = _quick_layer = _not_loaded


def new_rng(device, seed):
    """Device state of one random stream: int64[2] = {seed, calls so far} (the form of FusedTD3.new_rng)."""
    return torch.tensor([int(seed) & 0x7fffffffffffffff, 0], dtype=torch.long, device=device)


def advance(rng):
    """Move the stream on by one call, on the device: the next draw of every site is a new one."""
    rng[1:].add_(1)


def steps(p):
    """The probability as the masks hold it, in steps of 2^-16: elements whose 16 bits are below this are dropped."""
    return int(round(float(p) * 65536))


# ---- argument checks -------------------------------------------------------------------------------------------------------------------------
def _check_x(x):
    if not isinstance(x, torch.Tensor) or x.dtype not in DTYPES:
        raise TypeError("x has to be a float32, bfloat16 or float16 tensor, got %s" % (getattr(x, "dtype", type(x).__name__),))
    if x.layout != torch.strided or x.device.type not in ("cuda", "cpu"):
        raise TypeError("x has to be a dense tensor on a HIP device or the CPU")


def _check_draw(x, p, rng, site):
    """-> the threshold that the mask's 16-bit words are compared with (probability p in steps of 2^-16)."""
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError("p has to be in [0, 1], got %r" % p)
    if not isinstance(rng, torch.Tensor) or rng.dtype != torch.long or rng.shape != (2,) or rng.device != x.device or not rng.is_contiguous():
        raise ValueError("rng has to be a contiguous int64 tensor {seed, calls} on x's device (new_rng)")
    if not 0 <= int(site) < (1 << 31) - 16:
        raise ValueError("site has to be in [0, 2^31 - 16), got %r" % (site,))
    if x.numel() > MAX_DRAWN:
        raise ValueError("a mask has at most 2^35 elements, x has %d" % x.numel())
    return steps(p)


def _no_trace():
    """The plain form reads the random state on the host: a trace would hold its mask as a constant.  (Device tensors: csrc/regularise_torch.cpp refuses any kind of recording.)"""
    if torch.jit.is_tracing():
        raise RuntimeError("plen_ml_walk_amd.regularise cannot be traced: the trace would draw one mask for ever")


def _check_norm(x, groups, weight, bias, eps, act):
    if x.dim() < 2:
        raise ValueError("x has to be [N, C] or [N, ..., C], got %d dimension(s)" % x.dim())
    ch, groups = x.shape[-1], int(groups)
    if groups < 1 or ch < 1 or ch % groups:
        raise ValueError("groups (%d) has to divide the %d channels of x" % (groups, ch))
    long = math.prod(x.shape[1:-1]) > 1
    if ch > (MAX_C_LONG if long else MAX_C):
        raise ValueError("x has %d channels; at most %d are supported for [N, ..., C] and %d for [N, C]" % (ch, MAX_C_LONG, MAX_C))
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and (not isinstance(t, torch.Tensor) or t.shape != (ch,) or t.dtype not in DTYPES or t.device != x.device):
            raise ValueError("%s has to be a float tensor of x's %d channels on x's device" % (name, ch))
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError("weight and bias have to be of one type, got %s and %s" % (weight.dtype, bias.dtype))
    if not 0.0 < float(eps) < math.inf or C.c_float(float(eps)).value == 0.0:
        raise ValueError("eps has to be positive (a group whose elements are equal has no variance), got %r" % (eps,))
    if act not in ACTS:
        raise ValueError("act has to be one of %s, got %r" % (", ".join(ACTS), act))
    return groups


# ---- the definitions as elementary torch operations (CPU tensors) ----------------------------------------------------------------------------------
def _keep(shape, cut, rng, site):
    """The mask: Philox4x32-10 words of counter (element >> 3, calls, calls >> 32, 16 + site) and key = seed, as int64 tensors; 16 bits per element."""
    n, m = math.prod(shape), 0xFFFFFFFF
    seed, calls = (int(v) for v in rng.tolist())
    c0 = torch.arange((n + 7) // 8, device=rng.device)
    c1, c2, c3 = (torch.full_like(c0, v) for v in (calls & m, (calls >> 32) & m, 16 + site))
    k0, k1 = seed & m, (seed >> 32) & m
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57          # (the product may wrap into the sign bit: its 64 bits are what counts)
        c0, c1, c2, c3 = ((b >> 32) & m) ^ c1 ^ k0, b & m, ((a >> 32) & m) ^ c3 ^ k1, a & m
        k0, k1 = (k0 + 0x9E3779B9) & m, (k1 + 0xBB67AE85) & m
    w = torch.stack((c0, c1, c2, c3), 1)
    return (torch.stack((w & 0xFFFF, w >> 16), 2).view(-1)[:n] >= cut).view(shape)


def _scale(cut):
    return 65536.0 / (65536 - cut) if cut < 65536 else 0.0


def _plain_norm(x, groups, weight, bias, eps, act, keep, cut):
    xd = x.float()
    if keep is not None:
        xd = torch.where(keep, xd * _scale(cut), 0.0)
    xd = xd.reshape(x.shape[0], math.prod(x.shape[1:-1]), groups, x.shape[-1] // groups)
    mid = xd - xd.mean((1, 3), keepdim=True)
    z = (mid / torch.sqrt((mid * mid).mean((1, 3), keepdim=True) + eps)).reshape(x.shape)
    if weight is not None:
        z = z * weight.float()
    if bias is not None:
        z = z + bias.float()
    z = torch.relu(z) if act == "relu" else z * torch.sigmoid(z) if act == "silu" else z
    return z.to(x.dtype)


# ---- the operators ----------------------------------------------------------------------------------------------------------------------------------
def dropout(x, p, rng, site=0):
    """Each element of x is kept with probability 1 - p and scaled by 1 / (1 - p), or becomes 0 (whatever it held: a dropped NaN is 0).

    p is held in steps of 2^-16 (the scale is that of the step, so the expectation is exact); p = 1 drops everything.  x: float32, bfloat16 or
    float16, any shape of up to 2^35 elements; rng: {seed, calls} (`new_rng`), read and not advanced; site: the number of this place in the model.  Returns a
    contiguous tensor of x's type; the gradient with respect to x draws the same mask again.  Rows of contiguous elements a constant stride apart (a column
    slice) are read in place, other layouts are copied first."""
    y = _quick_dropout(x, p, rng, site)
    if y is not None:
        return y
    _check_x(x)
    cut, site = _check_draw(x, p, rng, site), int(site)
    if x.device.type == "cpu":
        _no_trace()
        return torch.where(_keep(x.shape, cut, rng, site), x.float() * _scale(cut), 0.0).to(x.dtype)
    return (_nodes or _load_nodes()).dropout(x, cut, rng, site)


def group_norm_act(x, groups, weight=None, bias=None, eps=1e-5, act="relu"):
    """act(group_norm(x) * weight + bias) over channels-last data: x [N, C] or [N, ..., C] (float32, bfloat16, float16), statistics over the positions and the
    C / groups neighbouring channels of each (n, group), act "none", "relu" or "silu"; groups = 1 with [N, C] is layer norm.

    weight, bias: [C] of one float type (it may differ from x's) or None.  Returns a contiguous tensor of x's type; differentiable (once) in x, weight and
    bias.  At most 8192 channels where there are positions, 32768 for [N, C].  Each x[n] has to be contiguous (the stride between them is free: a column slice of a
    wider matrix is read in place); what is laid out otherwise is copied first."""
    y = _quick_norm(x, groups, weight, bias, eps, act)
    if y is not None:
        return y
    _check_x(x)
    groups, eps = _check_norm(x, groups, weight, bias, eps, act), float(eps)
    if x.device.type == "cpu":
        return _plain_norm(x, groups, weight, bias, eps, act, None, 0)
    return (_nodes or _load_nodes()).norm(x, weight, bias, groups, eps, ACTS[act], 0, None, 0)


def dropout_norm_act(x, p, rng, groups, weight=None, bias=None, site=0, eps=1e-5, act="relu"):
    """act(group_norm(dropout(x)) * weight + bias) in one pass: `group_norm_act` of `dropout(x, p, rng, site)`, which is not rounded in between."""
    y = _quick_layer(x, p, rng, groups, weight, bias, site, eps, act)
    if y is not None:
        return y
    _check_x(x)
    cut, site = _check_draw(x, p, rng, site), int(site)
    groups, eps = _check_norm(x, groups, weight, bias, eps, act), float(eps)
    if x.device.type == "cpu":
        _no_trace()
        return _plain_norm(x, groups, weight, bias, eps, act, _keep(x.shape, cut, rng, site), cut)
    return (_nodes or _load_nodes()).norm(x, weight, bias, groups, eps, ACTS[act], cut, rng, site)
