"""Regularisation of the Q networks' hidden layers: dropout whose mask comes from the counter-based generator and is never stored, group norm
with an activation over channels-last data, and the two in one pass (linear -> dropout -> norm -> activation), each with its gradient.  HIP kernels of
csrc/regularise.hip behind the C ABI include/plenreg.h, bound with ctypes; td3.RegularisedCritic is the framework's own caller.

The twin critics' hidden rows lie side by side in one [B, 512] matrix, so group norm with two groups is both networks' layer norm in one call.

Random state: an int64[2] device tensor {seed, calls so far}, the form every draw of this package uses (`new_rng`).  Which mask a call draws depends
on that state, on `site` (one number per place in the model) and on the element's index alone, not on type, strides or launch shape.  A call only READS the
state; `advance` moves it on, once per iteration, as a kernel (so a captured graph draws new masks at every replay).  The backward pass draws the
forward's mask again from a 16-byte snapshot that the forward kernel takes.

CPU tensors take the same definitions as elementary torch operations (autograd differentiates them): the multi-process CPU path of td3.py."""
import ctypes as C
import math
import os

import torch
from torch.autograd.function import once_differentiable

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.environ.get("PLENREG_LIB") or os.path.join(_HERE, "csrc", "libplenreg.so")
EXPORTS = ["plenreg_dropout", "plenreg_norm_forward", "plenreg_norm_backward", "plenreg_norm_workspace", "plenreg_version"]
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ACTS = {"none": 0, "relu": 1, "silu": 2}
MAX_C, MAX_C_LONG = 32768, 8192           # PLENREG_MAX_C, PLENREG_MAX_C_LONG
MAX_DRAWN = 1 << 35                       # the mask counts blocks of 8 elements in 32 bits
_lib = None


class PlenRegError(RuntimeError):
    pass


class DropoutArgs(C.Structure):
    """Mirror of PlenRegDropout (include/plenreg.h)."""
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


def new_rng(device, seed):
    """Device state of one random stream: int64[2] = {seed, calls so far} (the form of FusedTD3.new_rng)."""
    return torch.tensor([int(seed) & 0x7fffffffffffffff, 0], dtype=torch.long, device=device)


def advance(rng):
    """Move the stream on by one call, on the device: the next draw of every site is a new one."""
    rng[1:].add_(1)


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
    return int(round(p * 65536))


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


def _launch(fn, args, device):
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            rc = fn(C.byref(args), torch.cuda.current_stream(device).cuda_stream)
    else:
        rc = fn(C.byref(args), torch.cuda.current_stream(device).cuda_stream)
    if rc != 0:
        raise PlenRegError("libplenreg kernel launch failed: HIP error %d" % -rc)


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


# ---- dropout --------------------------------------------------------------------------------------------------------------------------------------
def _rows(x):
    """x as rows of contiguous elements, a constant stride apart: (x, rows, cols, stride); what is laid out otherwise is copied first."""
    if x.is_contiguous():
        return x, 1, x.numel(), 0
    shape, stride = x.shape, x.stride()
    k = x.dim()
    want = 1
    while k and (stride[k - 1] == want or shape[k - 1] == 1):          # the contiguous dimensions at the end
        want *= shape[k - 1]
        k -= 1
    lead = [(s, st) for s, st in zip(shape[:k], stride[:k]) if s != 1]
    if want > 1 and all(a[1] == b[0] * b[1] for a, b in zip(lead, lead[1:])):
        return x, x.numel() // want, want, lead[-1][1] if lead else 0
    x = x.contiguous()
    return x, 1, x.numel(), 0


def _dropout_kernel(x, cut, rng, site, used=None):
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if x.numel():
        a = DropoutArgs()
        x, a.rows, a.cols, a.x_stride = _rows(x)
        a.x, a.y, a.rng, a.used = x.data_ptr(), y.data_ptr(), rng.data_ptr(), used.data_ptr() if used is not None else None
        a.dtype, a.cut, a.site = DTYPES[x.dtype], cut, site
        _launch(load().plenreg_dropout, a, x.device)
    elif used is not None:
        used.copy_(rng)
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, cut, rng, site):
        used = torch.empty_like(rng)
        y = _dropout_kernel(x, cut, rng, site, used)
        ctx.save_for_backward(used)
        ctx.cut, ctx.site = cut, site
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        return _dropout_kernel(dy, ctx.cut, ctx.saved_tensors[0], ctx.site), None, None, None


def dropout(x, p, rng, site=0):
    """Each element of x is kept with probability 1 - p and scaled by 1 / (1 - p), or becomes 0 (whatever it held: a dropped NaN is 0).

    p is held in steps of 2^-16 (the scale is that of the step, so the expectation is exact); p = 1 drops everything.  x: float32, bfloat16 or
    float16, any shape; rng: {seed, calls} (`new_rng`), read and not advanced; site: the number of this place in the model.  Returns a contiguous tensor of
    x's type; the gradient with respect to x draws the same mask again."""
    _check_x(x)
    cut, site = _check_draw(x, p, rng, site), int(site)
    if x.device.type == "cpu":
        return torch.where(_keep(x.shape, cut, rng, site), x.float() * _scale(cut), 0.0).to(x.dtype)
    if x.requires_grad and torch.is_grad_enabled():
        return _Dropout.apply(x, cut, rng, site)
    return _dropout_kernel(x, cut, rng, site)


# ---- group norm with an activation, with dropout before it or without ------------------------------------------------------------------------------
def _slabs(x):
    """x with the elements of each x[n] contiguous, and the distance of x[n] from x[n + 1]."""
    if not x.is_contiguous() and not x[0].is_contiguous():
        x = x.contiguous()
    return x, x.stride(0)


def _param(t, x):
    """A parameter in a type the kernels read beside x's: float32 or x's own."""
    return t if t is None or t.dtype == torch.float32 or t.dtype == x.dtype else t.float()


def _norm_args(x, groups, weight, bias, eps, act, cut, site):
    a = NormArgs()
    a.N, a.L, a.C, a.G = x.shape[0], math.prod(x.shape[1:-1]), x.shape[-1], groups
    a.dtype, a.act, a.cut, a.site, a.eps = DTYPES[x.dtype], ACTS[act], cut, site, eps
    for t in (weight, bias):
        if t is not None:
            a.w_dtype = DTYPES[t.dtype]
    a.w, a.b = weight.data_ptr() if weight is not None else None, bias.data_ptr() if bias is not None else None
    return a


def _workspace(a, backward, device):
    n = load().plenreg_norm_workspace(C.byref(a), backward)
    if n < 0:
        raise PlenRegError("libplenreg refuses these sizes: N %d, L %d, C %d, groups %d" % (a.N, a.L, a.C, a.G))
    ws = torch.empty(n, dtype=torch.uint8, device=device) if n else None
    a.ws = ws.data_ptr() if n else None
    return ws


def _norm_forward(x, groups, weight, bias, eps, act, cut, rng, site, stats=None, used=None):
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if x.numel():
        (x, stride), weight, bias = _slabs(x), _param(weight, x), _param(bias, x)
        a = _norm_args(x, groups, weight, bias, eps, act, cut, site)
        a.x, a.x_stride, a.out = x.data_ptr(), stride, y.data_ptr()
        a.stats = stats.data_ptr() if stats is not None else None
        if cut:
            a.rng, a.used = rng.data_ptr(), used.data_ptr() if used is not None else None
        ws = _workspace(a, 0, x.device)          # noqa: F841  (alive until the launch)
        _launch(load().plenreg_norm_forward, a, x.device)
    return y


class _NormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, act, cut, rng, site):
        stats = torch.empty(x.shape[0], groups, 2, dtype=torch.float64, device=x.device)
        used = torch.empty_like(rng) if cut else None
        y = _norm_forward(x, groups, weight, bias, eps, act, cut, rng, site, stats, used)
        ctx.save_for_backward(x, weight, bias, stats, used)
        ctx.rest = (groups, eps, act, cut, site)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, bias, stats, used = ctx.saved_tensors
        groups, eps, act, cut, site = ctx.rest
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        types = [t.dtype if t is not None else None for t in (weight, bias)]
        weight, bias = _param(weight, x), _param(bias, x)
        dw = torch.empty_like(weight) if ctx.needs_input_grad[1] else None
        db = torch.empty_like(bias) if ctx.needs_input_grad[2] else None
        if x.numel():
            (x, xs), (dy, dys) = _slabs(x), _slabs(dy)
            a = _norm_args(x, groups, weight, bias, eps, act, cut, site)
            a.x, a.x_stride, a.dy, a.dy_stride, a.out, a.stats = x.data_ptr(), xs, dy.data_ptr(), dys, dx.data_ptr(), stats.data_ptr()
            a.dw, a.db = dw.data_ptr() if dw is not None else None, db.data_ptr() if db is not None else None
            a.rng = used.data_ptr() if cut else None
            ws = _workspace(a, 1, x.device)      # noqa: F841  (alive until the launch)
            _launch(load().plenreg_norm_backward, a, x.device)
        else:
            for t in (dw, db):
                if t is not None:
                    t.zero_()
        dw, db = (t if t is None or t.dtype == dt else t.to(dt) for t, dt in zip((dw, db), types))
        return dx, dw, db, None, None, None, None, None, None


def _norm(x, groups, weight, bias, eps, act, cut, rng, site):
    weight, bias = (t.contiguous() if t is not None else None for t in (weight, bias))
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or (bias is not None and bias.requires_grad)):
        return _NormAct.apply(x, weight, bias, groups, eps, act, cut, rng, site)
    return _norm_forward(x, groups, weight, bias, eps, act, cut, rng, site)


def group_norm_act(x, groups, weight=None, bias=None, eps=1e-5, act="relu"):
    """act(group_norm(x) * weight + bias) over channels-last data: x [N, C] or [N, ..., C] (float32, bfloat16, float16), statistics over the positions and the
    C / groups neighbouring channels of each (n, group), act "none", "relu" or "silu"; groups = 1 with [N, C] is layer norm.

    weight, bias: [C] of one float type (it may differ from x's) or None.  Returns a contiguous tensor of x's type; differentiable in x, weight and
    bias.  At most 8192 channels where there are positions, 32768 for [N, C].  Each x[n] has to be contiguous (the stride between them is free: a column slice of a
    wider matrix is read in place); what is laid out otherwise is copied first."""
    _check_x(x)
    groups, eps = _check_norm(x, groups, weight, bias, eps, act), float(eps)
    if x.device.type == "cpu":
        return _plain_norm(x, groups, weight, bias, eps, act, None, 0)
    return _norm(x, groups, weight, bias, eps, act, 0, None, 0)


def dropout_norm_act(x, p, rng, groups, weight=None, bias=None, site=0, eps=1e-5, act="relu"):
    """act(group_norm(dropout(x)) * weight + bias) in one pass: `group_norm_act` of `dropout(x, p, rng, site)`, which is not rounded in between."""
    _check_x(x)
    cut, site = _check_draw(x, p, rng, site), int(site)
    groups, eps = _check_norm(x, groups, weight, bias, eps, act), float(eps)
    if x.device.type == "cpu":
        return _plain_norm(x, groups, weight, bias, eps, act, _keep(x.shape, cut, rng, site), cut)
    return _norm(x, groups, weight, bias, eps, act, cut, rng, site)
