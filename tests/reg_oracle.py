"""The regularisation operators' definitions in 64 bits (numpy masks, torch.float64 arithmetic on the CPU), and how far a 32-bit evaluation may be off.

Written apart from plen_ml_walk_amd/regularise.py and its kernels.  u = 2^-24 is half a step of float32, half(t) = finfo(t).eps / 2 that of a result's type."""
import math

import numpy as np
import torch

U = 2.0 ** -24


def philox(block, seed, calls, tag):
    """Philox4x32-10 in numpy uint64: block = array of counter words 0; -> four uint32 word arrays."""
    m = np.uint64(0xFFFFFFFF)
    block = np.asarray(block, dtype=np.uint64)
    c = [block & m] + [np.full_like(block, v) for v in (calls & 0xFFFFFFFF, (calls >> 32) & 0xFFFFFFFF, tag)]
    k = [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        s = np.uint64(32)
        c = [(b >> s) ^ c[1] ^ np.uint64(k[0]), b & m, (a >> s) ^ c[3] ^ np.uint64(k[1]), a & m]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def cut_of(p):
    return int(round(p * 65536))


def scale_of(p):
    c = cut_of(p)
    return 65536.0 / (65536 - c) if c < 65536 else 0.0


def keep_at(index, p, seed, calls, site):
    """Mask of the elements with these flat indices (int array)."""
    index = np.asarray(index, dtype=np.uint64)
    w = np.stack(philox(index >> np.uint64(3), seed, calls, 16 + site), -1)
    k = (index & np.uint64(7)).astype(np.int64)
    word = np.take_along_axis(w, (k >> 1)[..., None], -1)[..., 0]
    half = np.where(k & 1, word >> np.uint64(16), word & np.uint64(0xFFFF))
    return half >= np.uint64(cut_of(p))


def keep(shape, p, rng, site):
    seed, calls = (int(v) for v in rng.tolist())
    n = math.prod(shape)
    return torch.from_numpy(keep_at(np.arange(n), p, seed, calls, site)).view(shape) if n else torch.ones(shape, dtype=torch.bool)


def half(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half a step below the smallest normal value."""
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2


class Norm(object):
    """act(group_norm(dropout(x)) w + b) and its gradients in float64, with bounds on a 32-bit evaluation's error (arrays like the results)."""

    def __init__(self, x, groups, w, b, eps, act, mask=None, p=0.0, dy=None):
        dt = x.dtype
        x = x.detach().cpu().double()
        ch = x.shape[-1]
        self.shape = x.shape
        eps = float(np.float32(eps))
        four = (x.shape[0], -1, groups, ch // groups)
        w = torch.ones(ch, dtype=torch.float64) if w is None else w.detach().cpu().double()
        b = torch.zeros(ch, dtype=torch.float64) if b is None else b.detach().cpu().double()
        w, b = w.view(groups, -1), b.view(groups, -1)
        scale = scale_of(p) if mask is not None else 1.0
        xd = x if mask is None else torch.where(mask, x * scale, torch.zeros_like(x))
        xd = xd.reshape(four)
        mean = xd.mean((1, 3), keepdim=True)
        rstd = 1 / torch.sqrt(((xd - mean) ** 2).mean((1, 3), keepdim=True) + eps)
        xh = (xd - mean) * rstd
        z = xh * w + b
        s = torch.sigmoid(z)
        y = {"none": z, "relu": torch.relu(z), "silu": z * s}[act]
        # dropout's product, the difference from the mean and the product with rstd round once each, relative to operands of size |xd| + |mean|;
        # rstd itself is rounded once: 6 u covers them
        size = (xd.abs() + mean.abs()) * rstd
        e_xh = 6 * U * size
        e_z = e_xh * w.abs() + 2 * U * ((xh * w).abs() + b.abs())
        # |silu'| <= 1.1; exp's argument, exp, the sum and the quotient: (|z| + 8) u of the result
        e_y = 1.1 * e_z + (((z.abs() + 8) * U * y.abs()) if act == "silu" else 0)
        self.y = y.reshape(x.shape)
        self.y_tol = e_y.reshape(x.shape) + half(dt) * (self.y.abs() + e_y.reshape(x.shape)) + tiny(dt)
        self.stats = (mean, rstd)
        if dy is None:
            return
        wt = dt
        dy = dy.detach().cpu().double().reshape(four)
        slope = {"none": torch.ones_like(z), "relu": (z > 0).double(), "silu": s * (1 + z * (1 - s))}[act]
        dz = dy * slope
        # |silu''| <= 0.5; its evaluation: (|z| + 10) u of terms of size <= 1 + |z| s
        e_dz = dy.abs() * ((0.5 * e_z + (z.abs() + 10) * U * (1 + z.abs() * s)) if act == "silu" else 0) + 2 * U * dz.abs()
        gw = dz * w
        e_gw = e_dz * w.abs() + U * gw.abs()
        mean4 = lambda t: t.mean((1, 3), keepdim=True)  # noqa: E731
        m1, m2 = mean4(gw), mean4(gw * xh)
        # sums: at most 64 additions in a row before partial sums are joined in a tree (of at most 64 levels)
        e_m1 = mean4(e_gw) + 128 * U * mean4(gw.abs())
        e_m2 = mean4(e_gw * xh.abs() + gw.abs() * e_xh) + 128 * U * mean4((gw * xh).abs())
        dx = rstd * (gw - m1 - xh * m2)
        e_dx = rstd * (e_gw + e_m1 + xh.abs() * e_m2 + e_xh * m2.abs() + 8 * U * (gw.abs() + m1.abs() + (xh * m2).abs()))
        dx, e_dx = dx.reshape(x.shape) * scale, e_dx.reshape(x.shape) * scale
        if mask is not None:
            dx, e_dx = torch.where(mask, dx, torch.zeros_like(dx)), torch.where(mask, e_dx, torch.zeros_like(dx))
        self.dx = dx
        self.dx_tol = e_dx + half(dt) * (dx.abs() + e_dx) + tiny(dt)
        # parameter gradients: at most 512 additions in a row
        self.dw, self.db = (dz * xh).sum((0, 1)).reshape(-1), dz.sum((0, 1)).reshape(-1)
        self.dw_tol = (e_dz * xh.abs() + dz.abs() * e_xh + 600 * U * (dz * xh).abs()).sum((0, 1)).reshape(-1)
        self.db_tol = (e_dz + 600 * U * dz.abs()).sum((0, 1)).reshape(-1)


def inside(name, got, want, tol):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), name + ": NaN in other places"
    fine = torch.isfinite(want)
    off = (got - want).abs()[fine]
    bad = off > tol[fine]
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), name
    assert not bad.any(), "%s: %d of %d outside, worst %.3g against a bound of %.3g" % (
        name, int(bad.sum()), bad.numel(), float(off[bad].max()), float(tol[fine][bad][off[bad].argmax()]))
