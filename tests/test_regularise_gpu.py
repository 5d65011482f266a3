"""Regularisation operators on the GPU against their definitions in 64 bits (reg_oracle.py), at the sizes, layouts and values where they can go wrong."""
import itertools
import math

import numpy as np
import pytest
import torch

import reg_oracle as O
from plen_ml_walk_amd import regularise as R
from test_regularise_cpu import _refusals

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
ids = lambda v: str(v).replace("torch.", "")  # noqa: E731


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _rng(seed=0x123456789ABCDEF, calls=(3 << 32) + 9):
    return torch.tensor([seed, calls], device="cuda")


def _close_dropout(y, x, p, rng, site, name="y"):
    mask = O.keep(x.shape, p, rng, site)
    want = torch.where(mask, x.detach().cpu().double() * O.scale_of(p), 0.0)
    # the scale and the product in 32 bits, the result's own rounding
    O.inside(name, y, want, want.abs() * (2 * O.U + O.half(x.dtype) * (1 + 2 * O.U)) + O.tiny(x.dtype))


# ---- dropout ----------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9,), (63,), (100, 256), (3, 5, 7), (777, 1001), (64, 4096), (1, 1, 1), (2049, 3)], ids=ids)
def test_dropout_and_its_gradient(dtype, shape):
    x, dy = torch.randn(shape, generator=_gen(1)).to(dtype).cuda().requires_grad_(), torch.randn(shape, generator=_gen(2)).to(dtype).cuda()
    rng = _rng()
    for p in (0.01, 0.5):
        y = R.dropout(x, p, rng, site=3)
        assert y.dtype == dtype and y.is_contiguous()
        _close_dropout(y, x, p, rng, 3)
        (dx,) = torch.autograd.grad(y, x, dy)
        _close_dropout(dx, dy, p, rng, 3, "dx")
        with torch.no_grad():
            assert torch.equal(R.dropout(x, p, rng, site=3), y)


@pytest.mark.parametrize("p", [0.0, 2.0 ** -18, 2.0 ** -16, 1 - 2.0 ** -16, 1.0])
def test_dropout_at_the_ends_of_p(p):
    x = torch.randn(40001, generator=_gen(3)).cuda()
    y = R.dropout(x, p, _rng(), site=0)
    _close_dropout(y, x, p, _rng(), 0)
    if O.cut_of(p) == 0:
        assert torch.equal(x, y) and y.data_ptr() != x.data_ptr()
    if p == 1.0:
        assert not y.any()


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
def test_dropout_reads_any_layout(dtype):
    base = torch.randn(37, 90, generator=_gen(4)).to(dtype).cuda()
    big = torch.randn(6, 5, 4, 24, generator=_gen(5)).to(dtype).cuda()
    views = [base[:, 3:50], base[1:, 1:], base[::2, :88], base.t(), base[:, ::2], base[:, :1], base[:1, 5:], base[:1].expand(9, 90), base[:, :1].expand(37, 20), big[:, :, :, 1:],
             big[:, :, :2], big[::2], big.permute(1, 0, 2, 3), big[:, :1], base.reshape(-1)[1:], base.reshape(-1)[5:9]]
    for k, v in enumerate(views):
        _close_dropout(R.dropout(v, 0.3, _rng(), site=k), v, 0.3, _rng(), k, "view %d" % k)


def test_dropped_places_are_zero_whatever_they_held():
    x = torch.randn(4, 1000, generator=_gen(6)).cuda()
    mask = O.keep(x.shape, 0.4, _rng(), 1).cuda()
    for bad in (float("nan"), float("inf"), -float("inf")):
        z = torch.where(mask, x, torch.full_like(x, bad))
        assert torch.equal(R.dropout(z, 0.4, _rng(), site=1), R.dropout(x, 0.4, _rng(), site=1))
        args = (4, None, None, 1, 1e-5, "silu")
        assert torch.equal(R.dropout_norm_act(z, 0.4, _rng(), *args), R.dropout_norm_act(x, 0.4, _rng(), *args))
    z = torch.where(mask, torch.full_like(x, float("nan")), x)
    assert torch.equal(torch.isnan(R.dropout(z, 0.4, _rng(), site=1)), mask)


def test_dropout_past_32_bit_offsets():
    """4.5 G elements: rows that begin beyond 2^31 and 2^32 elements, mask blocks beyond 2^29."""
    rows, cols = 3, (3 << 29) + 5
    x = torch.empty(rows * cols, dtype=torch.float16, device="cuda").fill_(1.0).view(rows, cols)
    probe = [0, 1, cols - 3, cols, 2 * cols - 1, 2 * cols, (1 << 31) - 1, 1 << 31, (1 << 32) + 3, rows * cols - 9, rows * cols - 1]
    idx = np.concatenate([np.arange(max(0, i - 20), min(rows * cols, i + 20)) for i in probe])
    want = torch.from_numpy(O.keep_at(idx, 0.5, *(int(v) for v in _rng().tolist()), 3)).cuda()
    y = R.dropout(x, 0.5, _rng(), site=3).view(-1)
    assert torch.equal(y[torch.from_numpy(idx).cuda()], want.half() * 2)
    del y
    narrow = x[:, :1001]                                          # rows 1.6 G elements apart, read in place
    _close_dropout(R.dropout(narrow, 0.5, _rng(), site=3), narrow, 0.5, _rng(), 3)


# ---- group norm with an activation, with and without dropout -------------------------------------------------------------------------------
# (shape, groups): one element, groups of one element, odd channels, channels that do and do not fill a vector, one position and many, many slabs and one
SHAPES = [((1, 1), 1), ((3, 5), 5), ((5, 7), 1), ((4, 8), 1), ((100, 512), 2), ((9, 26), 2), ((33, 44), 1), ((5, 1001), 1), ((3, 1001), 7), ((2, 4096), 1), ((2, 4100), 2), ((3, 32768), 1),
          ((2, 20480), 1), ((300, 64), 8), ((1, 6), 3), ((700, 24), 3), ((2, 3, 8), 1), ((1, 2, 2), 1), ((3, 9, 12), 4), ((2, 33, 5, 13), 13), ((4, 17, 195), 13), ((1, 1000, 10), 2),
          ((2, 300, 320), 32), ((2, 64, 7), 1), ((600, 4, 32), 4), ((1, 5000, 3), 1), ((1, 70000, 8), 2), ((2, 40, 8192), 8), ((1, 3, 8185), 1), ((17, 2, 512), 2), ((2, 1500, 129), 3), ((200, 50, 40), 5)]


def _case(shape, groups, dtype, seed=7, wdtype=torch.float32):
    g = _gen(seed)
    ch = shape[-1]
    x = (torch.randn(shape, generator=g) * torch.exp(0.5 * torch.randn(ch, generator=g)) + torch.randn(ch, generator=g)).to(dtype).cuda().requires_grad_()
    dy = torch.randn(shape, generator=g).to(dtype).cuda()
    w, b = ((torch.randn(ch, generator=g) * s + m).to(wdtype).cuda().requires_grad_() for s, m in ((0.5, 1.0), (0.5, 0.0)))
    return x, dy, w, b


def _check(x, dy, w, b, groups, act, p, rng, site=2, eps=1e-5, exact_dx=True):
    drop = p is not None
    y = R.dropout_norm_act(x, p, rng, groups, w, b, site=site, eps=eps, act=act) if drop else R.group_norm_act(x, groups, w, b, eps=eps, act=act)
    assert y.dtype == x.dtype and y.is_contiguous() and y.shape == x.shape
    leaves = [t for t in (x, w, b) if t is not None]
    grads = dict(zip([n for n, t in (("dx", x), ("dw", w), ("db", b)) if t is not None], torch.autograd.grad(y, leaves, dy)))
    ref = O.Norm(x, groups, w, b, eps, act, O.keep(x.shape, p, rng, site) if drop else None, p or 0.0, dy)
    O.inside("y", y, ref.y, ref.y_tol)
    for name, got in grads.items():
        want, tol = getattr(ref, name), getattr(ref, name + "_tol")
        if name != "dx":
            assert got.dtype == (w if name == "dw" else b).dtype
            tol = tol + O.half(got.dtype) * (want.abs() + tol) + O.tiny(got.dtype)
        O.inside(name, got, want, tol)
    with torch.no_grad():
        again = R.dropout_norm_act(x, p, rng, groups, w, b, site=site, eps=eps, act=act) if drop else R.group_norm_act(x, groups, w, b, eps=eps, act=act)
        assert torch.equal(again.view(torch.uint8), y.view(torch.uint8))
    return y, grads


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("shape,groups", SHAPES, ids=ids)
def test_norm_and_its_gradients(shape, groups, dtype):
    x, dy, w, b = _case(shape, groups, dtype)
    acts = ["relu", "silu", "none"]
    for k, p in enumerate((None, 0.01, 0.4)):
        _check(x, dy, w, b, groups, acts[(k + len(shape) + groups) % 3], p, _rng())


@pytest.mark.parametrize("act", ["none", "relu", "silu"])
@pytest.mark.parametrize("shape,groups", [((64, 512), 2), ((3, 50, 24), 3), ((2, 3000, 64), 4)], ids=ids)
def test_every_activation_and_parameter_form(shape, groups, act):
    for dtype, wdtype, has_w, has_b in ((torch.float32, torch.float32, True, False), (torch.bfloat16, torch.bfloat16, True, True), (torch.float16, torch.float16, False, True),
                                        (torch.float32, torch.bfloat16, True, True), (torch.bfloat16, torch.float32, False, False)):
        x, dy, w, b = _case(shape, groups, dtype, wdtype=wdtype)
        for p in (None, 0.2):
            _check(x, dy, w if has_w else None, b if has_b else None, groups, act, p, _rng())


@pytest.mark.parametrize("shape,groups", [((6, 512), 2), ((3, 50, 24), 3), ((1, 40000, 16), 2)], ids=ids)
def test_groups_that_are_constant_or_wholly_dropped(shape, groups):
    """No variance: (x - mean) is zero, y = act(b), and nothing is infinite; the gradient is finite and small against 1 / sqrt(eps)."""
    for value in (0.0, 3.25, -1e6):
        for p in (None, 1.0):
            x = torch.full(shape, value, device="cuda", requires_grad=True)
            w, b = torch.randn(shape[-1], generator=_gen(8)).cuda().requires_grad_(), torch.randn(shape[-1], generator=_gen(9)).cuda().requires_grad_()
            dy = torch.randn(shape, generator=_gen(10)).cuda()
            y, grads = _check(x, dy, w, b, groups, "silu", p, _rng())
            assert torch.isfinite(y).all() and not grads["dw"].any()
            if p == 1.0:
                assert not grads["dx"].any()


@pytest.mark.parametrize("shape,groups", [((6, 512), 2), ((3, 50, 24), 3), ((1, 40000, 16), 2)], ids=ids)
def test_mean_far_from_zero(shape, groups):
    """Offsets 10^4 times the spread, where the square of the mean would swallow the variance in 32 bits; one outlier of 10^6 in another group."""
    x, dy, w, b = _case(shape, groups, torch.float32)
    with torch.no_grad():
        x += 1e4
        x[0].view(-1)[0] = 1e6
    for p in (None, 0.3):
        _check(x, dy, w, b, groups, "silu", p, _rng())


@pytest.mark.parametrize("shape,groups", [((6, 512), 2), ((3, 50, 24), 3), ((2, 40000, 16), 2)], ids=ids)
def test_nan_and_infinity_stay_in_their_group(shape, groups):
    for bad in (float("nan"), float("inf")):
        x, dy, w, b = _case(shape, groups, torch.float32)
        clean = R.group_norm_act(x, groups, w, b, act="relu").detach()
        with torch.no_grad():
            x[1].view(-1)[-1] = bad                     # slab 1, last group
        y = R.group_norm_act(x, groups, w, b, act="relu")
        d = shape[-1] // groups
        hit = torch.zeros(shape, dtype=torch.bool, device="cuda")
        hit[1, ..., -d:] = True
        assert torch.isnan(y[hit]).all() and torch.equal(y[~hit], clean[~hit])
        dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
        assert torch.isfinite(dx[~hit]).all() and torch.isfinite(dw[:-d]).all() and torch.isfinite(db[:-d]).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
def test_norm_reads_any_layout(dtype):
    """Column slices are read in place, everything else is copied first; expanded inputs and gradients count once per use."""
    g = _gen(11)
    rows = torch.randn(40, 600, generator=g).to(dtype).cuda()
    maps = torch.randn(5, 30, 48, generator=g).to(dtype).cuda()
    for v, groups in ((rows[:, 5:517], 2), (rows[:, 1:27], 2), (rows[::3, :512], 4), (rows[:1, :64].expand(40, 64), 1), (rows.t()[:64], 8), (rows[:, ::2], 3), (maps[:, 3:20], 4), (maps[:, :, :13], 1),
                      (maps.transpose(1, 2)[:, :, :24], 3), (maps[::2], 6), (maps[:1].expand(7, 30, 48), 2), (maps[:, :1].expand(5, 9, 48), 3), (rows.view(-1)[3:3 + 12 * 64].view(3, 4, 64), 2)):
        x = v.detach().requires_grad_()
        w, b = torch.randn(v.shape[-1], generator=g).cuda().requires_grad_(), torch.randn(v.shape[-1], generator=g).cuda().requires_grad_()
        wide = torch.randn(v.shape[:-1] + (v.shape[-1] + 3,), generator=g).to(dtype).cuda()
        for dy in (wide[..., 3:], wide[:1, ..., 1:-2].expand(v.shape), wide[..., :1].expand(v.shape)):
            _check(x, dy, w, b, groups, "relu", 0.2, _rng())
    # a leaf that is broadcast into the batch: its gradient is the sum over it
    leaf = torch.randn(1, 64, generator=g).cuda().requires_grad_()
    dy = torch.randn(40, 64, generator=g).cuda()
    (got,) = torch.autograd.grad(R.group_norm_act(leaf.expand(40, 64), 4, act="silu"), leaf, dy)
    ref = O.Norm(leaf.expand(40, 64), 4, None, None, 1e-5, "silu", dy=dy)
    O.inside("leaf", got, ref.dx.sum(0, keepdim=True), ref.dx_tol.sum(0, keepdim=True) + 40 * O.U * ref.dx.abs().sum(0, keepdim=True))


def test_norm_past_32_bit_offsets():
    """Slabs 1.6 G elements apart in a 3.2 G element buffer."""
    base = torch.empty(2, (3 << 29) + 7, dtype=torch.bfloat16, device="cuda")
    for shape, groups in (((2, 520), 4), ((2, 30, 24), 3), ((2, 30000, 24), 3)):
        x, dy, w, b = _case(shape, groups, torch.bfloat16)
        n = math.prod(shape[1:])
        v = base[:, -n:].view(shape) if len(shape) == 2 else base.as_strided(shape, (base.stride(0), shape[2], 1), base.shape[1] - n)
        with torch.no_grad():
            v.copy_(x)
        _check(v.detach().requires_grad_(), dy, w, b, groups, "silu", 0.1, _rng())


def test_norm_of_more_than_2_31_elements():
    """One slab of 2.2 G elements: its statistics and the ends of y and dx against 64-bit sums."""
    l, ch, groups = (1 << 27) + 3, 17, 1
    x = torch.empty(1, l, ch, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(1)).add_(1.0)
    with torch.no_grad():
        y = R.group_norm_act(x, groups, act="none")
        s = q = 0.0
        for part in x.view(-1).split(1 << 27):
            d = part.double()
            s += float(d.sum()); q += float((d * d).sum())
            del d
        mean = s / (l * ch)
        rstd = 1 / math.sqrt(q / (l * ch) - mean * mean + 1e-5)
        for at in (slice(0, 100), slice(l // 2, l // 2 + 100), slice(l - 100, l)):
            want = (x[0, at].cpu().double() - mean) * rstd
            O.inside("y", y[0, at], want, want.abs() * O.half(torch.bfloat16) * 1.01 + 20 * O.U)


def test_gradients_against_differences():
    """<dx, v> of the kernels against central differences of the 64-bit definition."""
    for shape, groups in (((6, 24), 2), ((2, 11, 10), 5)):
        x, dy, w, b = _case(shape, groups, torch.float32)
        for act in ("none", "silu", "relu"):
            mask = O.keep(shape, 0.3, _rng(), 2)
            y = R.dropout_norm_act(x, 0.3, _rng(), groups, w, b, site=2, act=act)
            for got, k in zip(torch.autograd.grad(y, (x, w, b), dy), range(3)):
                v = torch.randn(got.shape, generator=_gen(20 + k), dtype=torch.float64)
                at = [t.detach().cpu().double() for t in (x, w, b)]
                f = lambda s: float((O.Norm(*[at[0] + s * v if k == 0 else at[0]], groups, *[at[i] + s * v if k == i else at[i] for i in (1, 2)], 1e-5, act, mask, 0.3).y  # noqa: E731
                                     * dy.cpu().double()).sum())
                h = 1e-6
                diff, inner = (f(h) - f(-h)) / (2 * h), float((got.cpu().double() * v).sum())
                # differences of a 64-bit sum: ~1e-16 / h; the 32-bit gradient: 1e-5 of its size
                assert abs(diff - inner) <= 1e-6 + 1e-5 * float((got.cpu().double() * v).abs().sum()), (shape, act, k, diff, inner)


def test_empty_inputs_on_the_device():
    w = torch.randn(6, device="cuda", requires_grad=True)
    for shape in ((0, 6), (0, 3, 6), (4, 0, 6)):
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        for y in (R.group_norm_act(x, 2, w, w), R.dropout_norm_act(x, 0.5, _rng(), 2, w, w)):
            dx, dw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
            assert y.shape == dx.shape == shape and not dw.any()
        y = R.dropout(x, 0.5, _rng())
        assert torch.autograd.grad(y, x, torch.zeros_like(y))[0].shape == shape


def test_refusals_on_the_device():
    for kind, call in _refusals("cuda"):
        with pytest.raises(kind):
            call()
    x = torch.randn(4, 6, device="cuda")
    with pytest.raises(ValueError):
        R.dropout(x, 0.5, R.new_rng("cpu", 1))
    with pytest.raises(ValueError):
        R.group_norm_act(x, 2, torch.ones(6))


# ---- together, as a hidden layer uses them ---------------------------------------------------------------------------------------------------
def test_the_pass_in_one_is_dropout_then_norm():
    for dtype in DTYPES:
        x, dy, w, b = _case((64, 512), 2, dtype)
        one = R.dropout_norm_act(x, 0.1, _rng(), 2, w, b, site=5, act="relu")
        two = R.group_norm_act(R.dropout(x, 0.1, _rng(), site=5), 2, w, b, act="relu")
        # apart by the rounding of dropout's result to x's type, half a step of elements of size <= ~6 standard deviations, and y's own
        assert float((one.detach().float() - two.detach().float()).abs().max()) <= 40 * O.half(dtype) + 1e-5
        for p in (0.0, 2.0 ** -18):
            zero = R.dropout_norm_act(x, p, _rng(), 2, w, b, site=5, act="relu")
            assert torch.equal(zero, R.group_norm_act(x, 2, w, b, act="relu"))


def test_the_backward_pass_draws_the_forward_mask_after_the_state_moved_on():
    x, dy, w, b = _case((50, 64), 2, torch.float32)
    rng = _rng()
    before = rng.clone()
    y1 = R.dropout(x, 0.5, rng, site=1)
    y2 = R.dropout_norm_act(x, 0.5, rng, 2, w, b, site=2)
    R.advance(rng)
    assert rng.tolist() == [before[0].item(), before[1].item() + 1]
    rng.fill_(77)
    (d1,) = torch.autograd.grad(y1, x, dy)
    _close_dropout(d1, dy, 0.5, before, 1, "dx")
    (d2,) = torch.autograd.grad(y2, x, dy)
    assert not d2[~O.keep(x.shape, 0.5, before, 2).cuda()].any()


def test_captured_steps_draw_new_masks_and_equal_eager_ones():
    """Two layers, forward and backward and the stream's advance in one graph: every replay equals the eager step of the same state, with other work between the replays;
    a second graph of the same operators does not disturb the first."""
    x, dy, w, b = _case((96, 512), 2, torch.float32)
    m, dm, wm, bm = _case((2, 3000, 40), 4, torch.float32, seed=9)
    rng = R.new_rng("cuda", 31)

    def step():
        h = R.dropout_norm_act(R.dropout(x, 0.2, rng, site=0), 0.1, rng, 2, w, b, site=1, act="relu")
        k = R.group_norm_act(m, 4, wm, bm, act="silu")
        out = (h, k) + torch.autograd.grad((h, k), (x, w, b, m, wm, bm), (dy, dm))
        R.advance(rng)
        return tuple(t.detach() for t in out)

    want = [tuple(t.clone() for t in step()) for _ in range(5)]
    assert not torch.equal(want[0][0], want[1][0])
    rng.copy_(R.new_rng("cuda", 31))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    rng.copy_(R.new_rng("cuda", 31))
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            graphs.append((g, step()))
    rng.copy_(R.new_rng("cuda", 31))
    for k in range(5):
        g, out = graphs[k % 2]
        other = graphs[(k + 1) % 2][1]
        kept = [t.clone() for t in other]
        g.replay()
        torch.cuda.synchronize()
        for a, c in zip(out, want[k]):
            assert torch.equal(a, c)
        for a, c in zip(other, kept):
            assert torch.equal(a, c)
        junk = torch.randn(1 << 20, device="cuda").sum().item()          # the program's own work between replays
        assert math.isfinite(junk)


def test_results_do_not_depend_on_stream_or_repetition():
    x, dy, w, b = _case((3, 5000, 48), 3, torch.bfloat16)
    rows = _case((4096, 512), 2, torch.float32)

    def both():
        out = []
        for (xx, d, ww, bb), groups in (((x, dy, w, b), 3), (rows, 2)):
            y = R.dropout_norm_act(xx, 0.1, _rng(), groups, ww, bb, site=1)
            out += [y.detach()] + list(torch.autograd.grad(y, (xx, ww, bb), d))
        return out

    first = both()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for s in streams * 2:                                      # two calls at once
        with torch.cuda.stream(s):
            got.append(both())
    torch.cuda.synchronize()
    for other in got:
        for a, c in zip(first, other):
            assert torch.equal(a, c)


def test_saved_inputs_are_watched():
    """Changing an input in place between the passes is an error, not a wrong gradient."""
    x = torch.randn(8, 64, device="cuda")
    w = torch.ones(64, device="cuda", requires_grad=True)
    y = R.group_norm_act(x, 2, w)
    x.add_(1)
    with pytest.raises(RuntimeError):
        y.sum().backward()


def test_a_second_derivative_is_refused():
    x, dy, w, b = _case((8, 64), 2, torch.float32)
    for y in (R.group_norm_act(x, 2, w, b), R.dropout(x, 0.3, _rng())):
        (dx,) = torch.autograd.grad(y, x, dy, create_graph=True)
        with pytest.raises(RuntimeError):
            dx.sum().backward()


def test_gradients_reach_only_what_asks_for_them():
    x, dy, w, b = _case((40, 64), 2, torch.float32)
    full = torch.autograd.grad(R.group_norm_act(x, 2, w, b), (x, w, b), dy)
    fixed = [t.detach() for t in (x, w, b)]
    for k, leaf in enumerate((x, w, b)):
        args = [leaf if i == k else fixed[i] for i in range(3)]
        (got,) = torch.autograd.grad(R.group_norm_act(args[0], 2, args[1], args[2]), leaf, dy)
        assert torch.equal(got, full[k])
    # the same tensor as weight and bias: its gradient is the sum of both
    both = w.detach().clone().requires_grad_()
    (got,) = torch.autograd.grad(R.group_norm_act(x, 2, both, both, act="none"), both, dy)
    dx, dw, db = torch.autograd.grad(R.group_norm_act(x, 2, w, w.detach(), act="none"), (x, w), dy) + torch.autograd.grad(
        R.group_norm_act(x, 2, w.detach(), w, act="none"), w, dy)
    assert torch.equal(got, dw + db)


@pytest.mark.parametrize("kind", ["dropout", "norm", "layer"])
def test_a_second_backward_needs_the_graph_kept(kind):
    x, w, b = (t.cuda().requires_grad_() for t in (torch.randn(9, 40, generator=_gen(1)), torch.ones(40), torch.zeros(40)))
    rng = _rng()
    call = {"dropout": lambda: R.dropout(x, 0.3, rng), "norm": lambda: R.group_norm_act(x, 2, w, b), "layer": lambda: R.dropout_norm_act(x, 0.3, rng, 2, w, b)}[kind]
    leaves, dy = [x] if kind == "dropout" else [x, w, b], torch.randn(9, 40, generator=_gen(2)).cuda()
    y = call()
    first = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    for a, b_ in zip(first, torch.autograd.grad(y, leaves, dy)):
        assert torch.equal(a, b_)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y, leaves, dy)
    if kind != "dropout":          # (dropout keeps no input)
        y = call()
        with torch.no_grad():
            x.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(y, leaves, dy)


def test_gradients_of_one_leaf_at_a_time():
    x, w, b = (t.cuda().requires_grad_() for t in (torch.randn(9, 40, generator=_gen(1)), torch.randn(40, generator=_gen(3)), torch.randn(40, generator=_gen(4))))
    dy = torch.randn(9, 40, generator=_gen(2)).cuda()
    whole = torch.autograd.grad(R.group_norm_act(x, 2, w, b), (x, w, b), dy)
    for k, leaf in enumerate((x, w, b)):
        (got,) = torch.autograd.grad(R.group_norm_act(x, 2, w, b), leaf, dy)
        assert torch.equal(got, whole[k])
    for k in ((0, 1), (0, 2), (1, 2)):           # some of the inputs without a gradient, or not there
        args = [t if i in k else t.detach() for i, t in enumerate((x, w, b))]
        got = torch.autograd.grad(R.group_norm_act(args[0], 2, args[1], args[2]), [args[i] for i in k], dy)
        assert all(torch.equal(g, whole[i]) for g, i in zip(got, k))


def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fwad
    x = torch.randn(4, 8, generator=_gen(1)).cuda()
    with fwad.dual_level():
        dual = fwad.make_dual(x, torch.ones_like(x))
        for call in (lambda: R.dropout(dual, 0.5, _rng()), lambda: R.group_norm_act(dual, 2)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()


@pytest.mark.parametrize("shape,groups", [((40, 2, 8192), 4), ((3, 2, 8192), 1), ((2, 3, 4104), 27), ((700, 40, 448), 448), ((4, 1089, 195), 13), ((2, 4096, 64), 64), ((1, 4096, 512), 8),
                                          ((1, 4096, 512), 16), ((2, 700, 200), 200), ((5, 1100, 90), 45),
                                          ((600, 2, 4096), 4096), ((300, 2, 2504), 2504), ((3, 70, 4104), 513), ((2, 9, 8184), 3), ((2, 300, 5000), 25), ((260, 30, 512), 512), ((300, 1000, 40), 8)], ids=ids)
def test_statistics_joined_in_the_results_launch_or_in_one_of_their_own(shape, groups):
    """Few partial sums per slab and many; few workgroups per slab beside many channels; groups of one channel."""
    x, dy, w, b = _case(shape, groups, torch.bfloat16)
    _check(x, dy, w, b, groups, "relu", 0.1, _rng())
    _check(x, dy, None, None, groups, "silu", None, None)


def test_arguments_of_other_number_types_mean_the_same():
    """What the native checks do not take as it comes (whole numbers, numpy's, a step of p) goes through the checks in Python to the same result."""
    x, rng = torch.randn(6, 48, generator=_gen(1)).cuda(), _rng()
    w = torch.randn(48, generator=_gen(2)).cuda()
    assert torch.equal(R.dropout(x, 1, rng), R.dropout(x, 1.0, rng)) and torch.equal(R.dropout(x, np.float32(0.25), rng, np.int64(2)), R.dropout(x, 0.25, rng, 2))
    assert torch.equal(R.group_norm_act(x, np.int32(3), w, None, 1, "silu"), R.group_norm_act(x, 3, w, None, 1.0, "silu"))
    assert torch.equal(R.dropout_norm_act(x, 0, rng, 3.0, w, eps=np.float64(1e-3)), R.dropout_norm_act(x, 0.0, rng, 3, w, eps=1e-3))
    for p in (2.0 ** -17, 3 * 2.0 ** -17, 5 * 2.0 ** -17):                # half steps: rounded to even by both
        assert torch.equal(R.dropout(x, p, rng), R.dropout(x, np.float32(p), rng))


@pytest.mark.parametrize("shape,groups", [((6, 512), 4), ((3, 50, 24), 3), ((300, 3, 2), 2), ((1, 40000, 16), 4), ((2, 777, 195), 13), ((3, 700, 30), 10)], ids=ids)
@pytest.mark.parametrize("value", [0.0, 1.7, -123.456])
def test_constant_groups_beside_others(shape, groups, value):
    """A group without variance has exactly its value as its mean, whatever the other groups of its slab hold: y = act(b) (to b's product), gates of z = 0 are shut."""
    x, dy, w, b = _case(shape, groups, torch.float32)
    with torch.no_grad():
        v = x.view(shape[0], -1, groups, shape[-1] // groups)
        v[:, :, 1::2] = value
    for act in ("none", "relu", "silu"):
        y, grads = _check(x, dy, w, None, groups, act, None, None)
        assert not y.detach().view(v.shape)[:, :, 1::2].any() and not grads["dw"].view(groups, -1)[1::2].any()
        _check(x, dy, w, b, groups, act, None, None)
        if value == 0.0:
            _check(x, dy, w, None, groups, act, 0.3, _rng())


@pytest.mark.parametrize("shape,groups", [((300, 3, 2), 2), ((40, 2, 24), 3), ((300, 2, 2504), 313), ((50, 30), 10)], ids=ids)
def test_groups_that_the_mask_leaves_empty_beside_others(shape, groups):
    x, dy, w, b = _case(shape, groups, torch.float32)
    assert not O.keep(shape, 0.9, _rng(), 2).view(shape[0], -1, groups, shape[-1] // groups).any(3).any(1).all()          # some are
    for act in ("none", "relu", "silu"):
        _check(x, dy, w, None, groups, act, 0.9, _rng())
        _check(x, dy, w, b, groups, act, 0.9, _rng())


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("shape,groups", [((3, 4104), 1), ((2, 4097), 1), ((5, 8192), 1), ((300, 8200), 1), ((3, 16388), 2), ((7, 32768), 1), ((2, 32765), 1), ((2, 32768), 4), ((2100, 4112), 1)], ids=ids)
def test_rows_wider_than_a_workgroup_holds(shape, groups, dtype):
    x, dy, w, b = _case(shape, groups, dtype)
    for act, p in (("relu", 0.1), ("silu", None)):
        _check(x, dy, w, b, groups, act, p, _rng())
    _check(x, dy, None, b, groups, "none", 0.5, _rng())
    wide = torch.zeros(shape[0], shape[1] + 5, dtype=dtype, device="cuda")
    wide[:, 3:3 + shape[1]] = x.detach()
    part = wide[:, 3:3 + shape[1]].requires_grad_()
    y, z = R.group_norm_act(x, groups, w, b), R.group_norm_act(part, groups, w, b)
    assert torch.equal(y, z) and all(torch.equal(s, t) for s, t in zip(torch.autograd.grad(y, (x, w, b), dy), torch.autograd.grad(z, (part, w, b), dy)))


# ---- what one group holds is nothing to the others ---------------------------------------------------------------------------------------------
# slabs by one workgroup, split ones joined in the result's launch and before it, of chunks that hold one group, two and more
GROUPED = [((3, 50, 24), 3), ((3, 50, 30), 3), ((3, 50, 12), 4), ((300, 3, 2), 2), ((2, 20000, 16), 2),
           ((2, 4096, 320), 32), ((2, 777, 195), 13), ((2, 4096, 64), 64), ((2, 4096, 512), 16), ((40, 2, 4096), 4096), ((300, 1000, 40), 8), ((530, 2, 4098), 683)]


def _layer(x, dy, w, b, groups, act, p):
    """y, dx, dw, db with dropout (p) or without."""
    x, w, b = (t.detach().requires_grad_() for t in (x, w, b))
    y = R.group_norm_act(x, groups, w, b, act=act) if p is None else R.dropout_norm_act(x, p, _rng(), groups, w, b, site=2, act=act)
    return (y.detach(),) + torch.autograd.grad(y, (x, w, b), dy)


def _spoil_elements(shape, groups, p):
    """NaN and infinity as the first element of a slab, as the first channel of a group behind another, and as the last element: every other group's y, dx, dw and db are those of the
    clean input, to the bit."""
    d = shape[-1] // groups
    x, dy, w, b = _case(shape, groups, torch.float32)
    kept = torch.ones(shape, dtype=torch.bool) if p is None else O.keep(shape, p, _rng(), 2)
    first_kept = lambda g: int(kept[1].view(-1, groups, d)[:, g].reshape(-1).nonzero()[0])  # noqa: E731
    for act, bad in (("relu", float("nan")), ("silu", float("inf")), ("none", -float("inf"))):
        clean = _layer(x, dy, w, b, groups, act, p)
        for g, last in ((0, False), (1, False), (groups - 1, True)):
            spoilt = x.detach().clone()
            group = spoilt[1].view(-1, groups, d)[:, g]
            at = first_kept(g)
            if last:
                at = int(kept[1].view(-1, groups, d)[:, g].reshape(-1).nonzero()[-1])
            group[at // d, at % d] = bad
            if p is not None:          # (whatever a dropped place holds)
                drop = ~kept[1].view(-1, groups, d)[:, g].cuda()
                group[drop] = float("nan")
            hit = torch.zeros((shape[0], spoilt[0].numel() // shape[-1], groups, d), dtype=torch.bool, device="cuda")
            hit[1, :, g] = True
            hit, chan = hit.view(shape), hit.any(1).any(0).view(-1)
            got = _layer(spoilt, dy, w, b, groups, act, p)
            assert torch.isnan(got[0][hit]).all(), (act, g)
            for name, a, c, at in zip(("y", "dx", "dw", "db"), got, clean, (~hit, ~hit, ~chan, ~chan)):
                assert torch.equal(a[at], c[at]), (name, act, bad, g, last)


def _spoil_parameters(shape, groups):
    d = shape[-1] // groups
    x, dy, w, b = _case(shape, groups, torch.float32)
    for act in ("none", "silu"):
        clean = _layer(x, dy, w, b, groups, act, None)
        for which in (0, 1):
            for bad in (float("nan"), float("inf")):
                params = [w.detach().clone(), b.detach().clone()]
                params[which][d] = bad               # the first channel of the second group
                got = _layer(x, dy, params[0], params[1], groups, act, None)
                others = torch.ones(groups, d, dtype=torch.bool, device="cuda")
                others[1] = False
                others = others.view(-1)
                for name, a, c in zip(("y", "dx", "dw", "db"), got, clean):
                    assert torch.equal(a[..., others], c[..., others]), (name, act, which, bad)


@pytest.mark.parametrize("p", [None, 0.3])
@pytest.mark.parametrize("shape,groups", GROUPED, ids=ids)
def test_a_bad_element_spoils_its_own_group_only(shape, groups, p):
    _spoil_elements(shape, groups, p)


@pytest.mark.parametrize("shape,groups", GROUPED, ids=ids)
def test_a_bad_parameter_spoils_its_own_group_only(shape, groups):
    _spoil_parameters(shape, groups)


@pytest.mark.parametrize("shape,groups", GROUPED, ids=ids)
def test_groups_of_quite_different_sizes(shape, groups):
    """The first group of each slab far away (an offset of 3e8, then 1e9 in its first element alone): the others keep their variance (64-bit sums around a value of another group would lose it)."""
    x, dy, w, b = _case(shape, groups, torch.float32)
    d = shape[-1] // groups
    for p in (None, 0.3):
        for far, part in ((3e8, slice(0, None)), (1e9, slice(0, 1))):
            z = x.detach().clone()
            group = z.view(shape[0], -1, groups, d)[:, :, 0]
            if part.stop is None:
                group += far
            else:
                group[:, 0, 0] = far
            _check(z.requires_grad_(), dy, w, b, groups, "silu", p, _rng())


# rows in whole and in partial chunks, and rows wider than a workgroup holds
ROW_GROUPED = [((6, 512), 4), ((9, 26), 2), ((5, 3003), 3), ((300, 30), 10), ((2, 10002), 2), ((3, 24600), 3), ((3, 24603), 3)]


@pytest.mark.parametrize("p", [None, 0.3])
@pytest.mark.parametrize("shape,groups", ROW_GROUPED, ids=ids)
def test_a_bad_element_of_a_row_spoils_its_own_group_only(shape, groups, p):
    _spoil_elements(shape, groups, p)


@pytest.mark.parametrize("shape,groups", ROW_GROUPED, ids=ids)
def test_a_bad_parameter_of_a_row_spoils_its_own_group_only(shape, groups):
    _spoil_parameters(shape, groups)


@pytest.mark.parametrize("shape,groups", ROW_GROUPED, ids=ids)
def test_groups_of_a_row_of_quite_different_sizes(shape, groups):
    x, dy, w, b = _case(shape, groups, torch.float32)
    with torch.no_grad():
        x.view(shape[0], groups, -1)[:, 0] += 3e8
    for p in (None, 0.3):
        _check(x, dy, w, b, groups, "silu", p, _rng())


# ---- a mean far above the spread, in 16 bits ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("shape,groups", [((4, 512), 2), ((4, 8008), 1), ((4, 4011), 3), ((2, 20008), 1), ((3, 100, 80), 2), ((3, 200, 39), 3), ((2, 20000, 16), 2), ((2, 4096, 30), 3), ((2, 3000, 48), 2)], ids=ids)
def test_few_elements_a_step_above_a_large_mean(shape, groups, dtype):
    """Elements of 1000 (and of -1000), few of them a step of the type higher: the mean lies between two steps, and what separates most elements from it is far below both.  x - mean rounds once, relative to
    itself; what the mean's first 24 bits leave out, below 2^-25 of it, is known to 24 bits of its own: e = 4 u |xh| + 2^-48 |mean| rstd before weight and bias (one rounding each, u of
    the value), sums of a group in 64 bits."""
    step = {torch.float32: 2.0 ** -13, torch.bfloat16: 4.0, torch.float16: 0.5}[dtype]
    d = shape[-1] // groups
    for sign in (1.0, -1.0):
        g = _gen(31)
        up = torch.rand(shape, generator=g) < 0.001
        up.view(shape[0], -1, groups, d)[:, 0, :, 0] = True
        x = (sign * (1000.0 + step * up)).to(dtype)
        assert int((x.abs() > 1000).sum()) == int(up.sum())
        w, b = torch.randn(shape[-1], generator=g) * 0.5 + 1, torch.randn(shape[-1], generator=g) * 0.5
        for weight, bias in ((None, None), (w, b)):
            y = R.group_norm_act(x.cuda(), groups, None if weight is None else weight.cuda(), None if bias is None else bias.cuda(), eps=1e-9, act="none")
            ref = O.Norm(x, groups, weight, bias, 1e-9, "none")
            mean, rstd = ref.stats
            xh = ((x.double().view(shape[0], -1, groups, d) - mean) * rstd)
            e = 4 * O.U * xh.abs() + 2.0 ** -48 * mean.abs() * rstd
            e, xh = e.view(shape), xh.view(shape)
            if weight is not None:
                e = e * weight.double().abs() + 2 * O.U * ((xh * weight.double()).abs() + bias.double().abs())
            O.inside("y", y, ref.y, e + O.half(dtype) * (ref.y.abs() + e) + O.tiny(dtype))


# ---- parameter gradients over very many slabs ----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("shape,groups", [((1 << 21, 2, 8), 1), ((1 << 20, 2, 6), 2), ((9000, 520, 8), 1), ((9000, 420, 10), 2), ((70000, 3, 5), 1), ((4097, 2, 4104), 3)], ids=ids)
def test_parameter_gradients_over_very_many_slabs(shape, groups):
    """Gradients all alike, so that 32-bit sums round the same way each time.  Each dz xh is off by (6 + 1) u and what xh itself is off by (as in the oracle), and its sums are in 64 bits over
    the slabs of a workgroup, rounded once, then in 64 bits again: 2 u of the sum of sizes."""
    g = torch.Generator("cuda").manual_seed(5)
    x = torch.randn(shape, device="cuda", generator=g)
    w, b = torch.ones(shape[-1], device="cuda", requires_grad=True), torch.zeros(shape[-1], device="cuda", requires_grad=True)
    dy = torch.full(shape, 1.0001, device="cuda")
    y = R.group_norm_act(x, groups, w, b, act="none")
    dw, db = torch.autograd.grad(y, (w, b), dy)
    want = dy[0, 0, 0].item() * shape[0] * shape[1]
    assert float((db.double() - want).abs().max()) <= 2 * O.U * want
    total, bound = torch.zeros(2, shape[-1], dtype=torch.float64, device="cuda")
    for part in x.split(max(1, (1 << 24) // (shape[1] * shape[2]))):
        v = part.double().view(part.shape[0], -1, groups, shape[-1] // groups)
        mean = v.mean((1, 3), keepdim=True)
        rstd = 1 / torch.sqrt(((v - mean) ** 2).mean((1, 3), keepdim=True) + float(np.float32(1e-5)))
        xh = ((v - mean) * rstd).reshape(part.shape)
        size = ((v.abs() + mean.abs()) * rstd).reshape(part.shape)
        total += (xh * dy[0, 0, 0].double()).sum((0, 1))
        bound += ((6 * O.U * size + 3 * O.U * xh.abs()) * dy[0, 0, 0].double()).sum((0, 1))
    assert bool(((dw.double() - total).abs() <= bound + O.U * total.abs()).all())


@pytest.mark.parametrize("kind", ["dropout", "norm", "layer"])
def test_calls_are_not_recorded(kind):
    from test_regularise_cpu import recorded_calls
    x, dy, w, b = _case((8, 64), 2, torch.float32)
    rng = _rng()
    call = {"dropout": lambda v: R.dropout(v, 0.3, rng), "norm": lambda v: R.group_norm_act(v, 2, w, b), "layer": lambda v: R.dropout_norm_act(v, 0.3, rng, 2, w, b)}[kind]
    want = call(x)                                       # (the first call loads the library; the next ones take the short way in)
    for name, run in recorded_calls(x.detach(), call):
        with pytest.raises(RuntimeError, match="plen_ml_walk_amd.regularise"):
            run()
    with pytest.raises(RuntimeError, match="plen_ml_walk_amd.regularise"):
        torch.autograd.grad(want, x, dy[None].expand(3, *dy.shape), is_grads_batched=True, retain_graph=True)
    assert torch.equal(call(x), want)


def test_views_whose_memory_holds_the_negatives():
    """The imaginary part of a conjugate is such a view; every tensor of a call may be one."""
    rng = _rng()
    one = torch.imag(torch.tensor([1.0 + 2.0j], device="cuda").conj())
    assert one.is_neg() and R.dropout(one, 0.0, rng).item() == -2.0
    x, dy, w, b = (t.detach() for t in _case((9, 48), 3, torch.float32))
    neg = lambda t: torch._neg_view(-t)  # noqa: E731
    assert neg(x).is_neg() and torch.equal(neg(x), x)
    for call in (lambda x, w, b, r: R.dropout(x, 0.3, r), lambda x, w, b, r: R.group_norm_act(x, 3, w, b), lambda x, w, b, r: R.dropout_norm_act(x, 0.3, r, 3, w, b)):
        for grad in (False, True):
            leaf = x.clone().requires_grad_(grad)
            want, got = call(leaf, w, b, rng), call(neg(leaf), neg(w), neg(b), neg(rng))
            assert torch.equal(want, got)
            if grad:
                (a,), (c,) = torch.autograd.grad(want, leaf, dy), torch.autograd.grad(got, leaf, neg(dy))
                assert torch.equal(a, c)


@pytest.mark.parametrize("shape,groups", GROUPED + ROW_GROUPED, ids=ids)
def test_a_bad_gradient_spoils_its_own_group_only(shape, groups):
    """NaN and infinity in dy at the first channel of a group behind another, and at the last element: dx of every other group, dw and db of every other channel are those of the clean gradient."""
    d = shape[-1] // groups
    x, dy, w, b = _case(shape, groups, torch.float32)
    for act, p, bad in (("silu", None, float("nan")), ("relu", 0.3, float("inf")), ("none", None, -float("inf"))):
        clean = _layer(x, dy, w, b, groups, act, p)
        for g, at in ((1, (0, 0)), (groups - 1, (-1, -1))):
            spoilt = dy.clone()
            spoilt[1].view(-1, groups, d)[:, g][at] = bad
            hit = torch.zeros((shape[0], dy[0].numel() // shape[-1], groups, d), dtype=torch.bool, device="cuda")
            hit[1, :, g] = True
            chan = torch.zeros(groups, d, dtype=torch.bool, device="cuda")
            chan[g, at[1]] = True
            got = _layer(x, spoilt, w, b, groups, act, p)
            for name, a, c, rest in zip(("y", "dx", "dw", "db"), got, clean, (torch.ones_like(hit).view(shape), ~hit.view(shape), ~chan.view(-1), ~chan.view(-1))):
                assert torch.equal(a[rest], c[rest]), (name, act, bad, g)


@pytest.mark.parametrize("shape,groups", [((4000, 9), 1), ((3000, 27), 3), ((500, 49), 1), ((60, 1001), 7), ((40, 3003), 1), ((3, 9001), 1), ((900, 3, 5), 1), ((300, 7, 30), 3), ((40, 11, 24), 3), ((2, 3001, 10), 2), ((2, 9001, 24), 3),
                                          ((4, 4003, 7), 7)], ids=ids)
def test_elements_that_are_their_groups_mean(shape, groups):
    """Whole numbers, one of each group set so that another of its elements is exactly the mean (counts without a power of two): its normalised value is 0, and without a bias its ReLU is shut.  The sums are exact in
    64 bits, so the mean has to be the quotient to its last bit."""
    d = shape[-1] // groups
    x, dy, w, _ = _case(shape, groups, torch.float32)
    v = torch.randint(-500, 500, shape, generator=_gen(41)).double()
    flat = v.view(shape[0], -1, groups, d).permute(0, 2, 1, 3).reshape(shape[0] * groups, -1)
    n = flat.shape[1]
    assert n & (n - 1)
    flat[:, 1] = torch.randint(-3, 4, (flat.shape[0],), generator=_gen(42)).double()          # (small, so that the last one stays within 24 bits)
    flat[:, -1] += n * flat[:, 1] - flat.sum(1)                  # the sum is n times element 1
    v = flat.view(shape[0], groups, -1, d).permute(0, 2, 1, 3).reshape(shape)
    x = v.float()
    assert torch.equal(x.double(), v)
    ref = O.Norm(x, groups, w, None, 1e-5, "none")
    tie = (ref.y == 0).view(shape[0], -1, groups, d)
    assert tie.any(3).any(1).all()                               # the oracle has them too
    for offset in (0.0, 4096.0):
        _check((x + offset).cuda().requires_grad_(), dy, w, None, groups, "relu", None, _rng())
