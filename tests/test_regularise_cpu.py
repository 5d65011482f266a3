"""Regularisation operators without a GPU: the library's boundary, the mask's definition, the CPU forms, and every refusal."""
import ctypes as C
import os
import re
import subprocess

import numpy as np
import pytest
import torch

import reg_oracle as O
from plen_ml_walk_amd import regularise as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    from plen_ml_walk_amd.build import build_regularise
    build_regularise()
    return R.load()


def test_library_exports_its_header(lib):
    hdr = open(os.path.join(ROOT, "include", "plenreg.h")).read()
    names = sorted(set(re.findall(r"\b(plenreg_[a-z0-9_]+)\s*\(", hdr)))
    assert sorted(R.EXPORTS) == names
    assert b"gfx950" in lib.plenreg_version()


def test_no_kernel_uses_scratch_memory(lib):
    """The compiler's report of the build: a spilling variant of the wide backward pass has given wrong results on lanes that a divergent branch leaves out."""
    import json
    from plen_ml_walk_amd.build import REG_RESOURCES
    report = json.load(open(REG_RESOURCES))
    assert len(report) > 30
    for name, r in report.items():
        assert r["ScratchSize"] == 0 and r.get("VGPRs Spill", 0) == 0 and r["LDS Size"] <= 65536, (name, r)


def test_struct_layouts_match_the_header(tmp_path):
    """Sizes and offsets of the ctypes mirrors against the C compiler's."""
    src = tmp_path / "s.c"
    lines = []
    for cname, mirror in (("PlenRegDropout", R.DropoutArgs), ("PlenRegNorm", R.NormArgs)):
        lines.append('printf("%%zu\\n", sizeof(%s));' % cname)
        lines += ['printf("%%zu\\n", offsetof(%s, %s));' % (cname, f[0]) for f in mirror._fields_]
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "plenreg.h"\nint main(void) { %s return 0; }\n' % " ".join(lines))
    exe = str(tmp_path / "s")
    subprocess.check_call(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), "-o", exe, str(src)])
    got = [int(v) for v in subprocess.check_output([exe]).split()]
    want = []
    for mirror in (R.DropoutArgs, R.NormArgs):
        want += [C.sizeof(mirror)] + [getattr(mirror, f[0]).offset for f in mirror._fields_]
    assert got == want


def test_generator_against_its_published_vectors():
    """Known answers of Philox4x32-10 (Random123's test vectors), for the oracle that everything else is held to."""
    z = O.philox([0], 0, 0, 0)
    assert [int(v[0]) for v in z] == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    f = O.philox([0xffffffff], 0xffffffffffffffff, 0xffffffffffffffff, 0xffffffff)
    assert [int(v[0]) for v in f] == [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]
    pi = O.philox([0x243f6a88], (0x299f31d0 << 32) | 0xa4093822, (0x13198a2e << 32) | 0x85a308d3, 0x03707344)
    assert [int(v[0]) for v in pi] == [0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1]


@pytest.mark.parametrize("p", [0.0, 2.0 ** -18, 0.005, 0.3, 0.5, 1 - 2.0 ** -16, 1.0])
@pytest.mark.parametrize("shape", [(1,), (13,), (3, 5, 7), (100, 256)])
def test_cpu_dropout_is_the_definition(p, shape):
    g = torch.Generator().manual_seed(1)
    rng = torch.tensor([0x123456789ABCDEF, (7 << 32) + 5])
    x = torch.randn(shape, generator=g).requires_grad_()
    y = R.dropout(x, p, rng, site=4)
    mask = O.keep(shape, p, rng, 4)
    want = torch.where(mask, x.detach().double() * O.scale_of(p), 0.0)
    O.inside("y", y, want, want.abs() * 2 * O.U)
    y.backward(torch.ones_like(y))
    O.inside("dx", x.grad, mask.double() * O.scale_of(p), torch.full(shape, 2 * O.U).double() * O.scale_of(p))


def test_masks_of_sites_calls_and_seeds_differ():
    x = torch.ones(4096)
    rng = R.new_rng("cpu", 11)
    a = R.dropout(x, 0.5, rng, site=0)
    assert torch.equal(a, R.dropout(x, 0.5, rng, site=0)) and rng.tolist() == [11, 0]
    b = R.dropout(x, 0.5, rng, site=1)
    R.advance(rng)
    assert rng.tolist() == [11, 1]
    c, d = R.dropout(x, 0.5, rng, site=0), R.dropout(x, 0.5, R.new_rng("cpu", 12), site=0)
    for u, v in ((a, b), (a, c), (a, d), (b, c)):
        # independent fair bits agree in 2048 +- 32 of 4096 places: six standard deviations
        assert abs(int(((u != 0) == (v != 0)).sum()) - 2048) < 6 * 32
    # 4096 draws kept with probability 1/2
    assert abs(int((a != 0).sum()) - 2048) < 6 * 32


@pytest.mark.parametrize("act", ["none", "relu", "silu"])
@pytest.mark.parametrize("shape,groups", [((5, 12), 3), ((3, 4, 5, 6), 2), ((2, 1, 8), 8), ((4, 7, 5), 1)])
@pytest.mark.parametrize("drop", [False, True])
def test_cpu_norm_is_the_definition(act, shape, groups, drop):
    g = torch.Generator().manual_seed(2)
    x, dy = torch.randn(shape, generator=g).requires_grad_(), torch.randn(shape, generator=g)
    w, b = torch.randn(shape[-1], generator=g).requires_grad_(), torch.randn(shape[-1], generator=g).requires_grad_()
    rng = R.new_rng("cpu", 5)
    y = R.dropout_norm_act(x, 0.25, rng, groups, w, b, site=2, act=act) if drop else R.group_norm_act(x, groups, w, b, act=act)
    y.backward(dy)
    ref = O.Norm(x, groups, w, b, 1e-5, act, O.keep(shape, 0.25, rng, 2) if drop else None, 0.25, dy)
    O.inside("y", y, ref.y, ref.y_tol)
    if shape != (2, 1, 8):          # (a group of one element: its gradient is what cancellation leaves)
        for name, got in (("dx", x.grad), ("dw", w.grad), ("db", b.grad)):
            O.inside(name, got, getattr(ref, name), getattr(ref, name + "_tol") + 64 * O.U)


def test_oracle_gradient_against_differences():
    """The oracle's own gradient formula against central differences of its forward pass, in 64 bits."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(3, 4, 6, generator=g, dtype=torch.float64)
    w, b, dy = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((6,), (6,), (3, 4, 6)))
    mask = torch.rand(3, 4, 6, generator=g) > 0.3
    f = lambda x, w, b, act: float((O.Norm(x, 2, w, b, 1e-5, act, mask, 0.3).y * dy).sum())  # noqa: E731
    for act in ("none", "silu", "relu"):
        ref = O.Norm(x, 2, w, b, 1e-5, act, mask, 0.3, dy)
        for name, at in (("dx", x), ("dw", w), ("db", b)):
            v = torch.randn(at.shape, generator=g, dtype=torch.float64)
            h = 1e-6
            put = lambda s: {"x": x, "w": w, "b": b, "act": act, name[1]: at + s * h * v}  # noqa: E731
            diff = (f(**put(1)) - f(**put(-1))) / (2 * h)
            want = float((getattr(ref, name) * v).sum())
            assert abs(diff - want) < 1e-7 * max(1.0, abs(want)), (act, name, diff, want)


def test_empty_inputs():
    w = torch.randn(6, requires_grad=True)
    for shape in ((0, 6), (0, 3, 6), (4, 0, 6)):
        x = torch.zeros(shape, requires_grad=True)
        y = R.group_norm_act(x, 2, w, None)
        assert y.shape == shape
    assert R.dropout(torch.zeros(0, 5), 0.5, R.new_rng("cpu", 1)).shape == (0, 5)


def _refusals(dev):
    x, rng, w = torch.randn(4, 6, device=dev), R.new_rng(dev, 1), torch.ones(6, device=dev)
    yield TypeError, lambda: R.dropout([1.0], 0.5, rng)
    yield TypeError, lambda: R.dropout(x.double(), 0.5, rng)
    yield TypeError, lambda: R.dropout(x.long(), 0.5, rng)
    for p in (-0.1, 1.1, float("nan")):
        yield ValueError, lambda p=p: R.dropout(x, p, rng)
    for bad in (None, rng.int(), rng[:1], torch.zeros(4, dtype=torch.long, device=dev)[::2], [1, 2]):
        yield ValueError, lambda bad=bad: R.dropout(x, 0.5, bad)
    for site in (-1, 1 << 31):
        yield ValueError, lambda site=site: R.dropout(x, 0.5, rng, site=site)
        yield ValueError, lambda site=site: R.dropout_norm_act(x, 0.5, rng, 2, site=site)
    yield ValueError, lambda: R.dropout(x[:1, :1].expand(1 << 18, (1 << 17) + 1), 0.5, rng)
    yield TypeError, lambda: R.group_norm_act(x.double(), 2)
    for groups in (0, -2, 4, 7):
        yield ValueError, lambda groups=groups: R.group_norm_act(x, groups)
    yield ValueError, lambda: R.group_norm_act(x[0], 2)
    yield ValueError, lambda: R.group_norm_act(x[:, :0], 1)
    yield ValueError, lambda: R.group_norm_act(x[:, :1].expand(4, 32769), 1)
    yield ValueError, lambda: R.group_norm_act(x[:, None, :1].expand(4, 2, 8193), 1)
    for bad in (w[:5], w.double(), w[None], 1.0):
        yield ValueError, lambda bad=bad: R.group_norm_act(x, 2, bad)
        yield ValueError, lambda bad=bad: R.group_norm_act(x, 2, None, bad)
    yield ValueError, lambda: R.group_norm_act(x, 2, w, w.half())
    for eps in (0.0, -1e-5, float("nan"), float("inf"), 1e-60):
        yield ValueError, lambda eps=eps: R.group_norm_act(x, 2, eps=eps)
    for act in ("tanh", None, 1):
        yield ValueError, lambda act=act: R.group_norm_act(x, 2, act=act)


def test_refusals_of_the_python_surface():
    n = 0
    for kind, call in _refusals("cpu"):
        with pytest.raises(kind):
            call()
        n += 1
    assert n > 35


def test_refusals_of_the_c_entries(lib):
    """Bad arguments come back as hipErrorInvalidValue before anything is launched (so this needs no GPU)."""
    bad = -1
    assert lib.plenreg_dropout(None, None) == lib.plenreg_norm_forward(None, None) == lib.plenreg_norm_backward(None, None) == bad
    assert lib.plenreg_norm_workspace(None, 0) < 0

    def drop(**kw):
        a = R.DropoutArgs(x=16, y=16, rng=16, rows=4, cols=6, x_stride=6, dtype=0, cut=100, site=0)
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.plenreg_dropout(C.byref(a), None)

    for kw in (dict(x=None), dict(y=None), dict(rng=None), dict(rows=0), dict(cols=0), dict(rows=-1), dict(x_stride=-1), dict(dtype=3), dict(dtype=-1),
               dict(cut=65537), dict(site=-1), dict(rows=1 << 34), dict(rows=1 << 40, cols=1 << 40)):
        assert drop(**kw) == bad, kw

    def norm(entry, **kw):
        a = R.NormArgs(x=16, dy=16, out=16, stats=16, dw=16, db=16, ws=16, rng=16, N=4, L=2, C=6, G=2, x_stride=12, dy_stride=12, eps=1e-5)
        for k, v in kw.items():
            setattr(a, k, v)
        return entry(C.byref(a), None) if entry is not lib.plenreg_norm_workspace else entry(C.byref(a), 1)

    shared = (dict(N=0), dict(L=0), dict(C=0), dict(G=0), dict(G=4), dict(G=-2), dict(dtype=3), dict(w_dtype=-1), dict(act=3), dict(act=-1), dict(eps=0.0), dict(eps=float("nan")),
              dict(cut=65537), dict(cut=1, site=-1), dict(C=8194), dict(L=1, C=32770), dict(L=1 << 60), dict(N=1 << 60), dict(N=1 << 31), dict(L=1 << 37, N=1 << 10))
    for entry in (lib.plenreg_norm_forward, lib.plenreg_norm_backward, lib.plenreg_norm_workspace):
        for kw in shared:
            assert norm(entry, **kw) < 0, kw
    for kw in (dict(x=None), dict(out=None), dict(x_stride=-1), dict(cut=1, rng=None)):
        assert norm(lib.plenreg_norm_forward, **kw) == norm(lib.plenreg_norm_backward, **kw) == bad, kw
    for kw in (dict(dy=None), dict(stats=None), dict(dy_stride=-1)):
        assert norm(lib.plenreg_norm_backward, **kw) == bad, kw


def test_missing_library_is_an_error(monkeypatch):
    monkeypatch.setattr(R, "_lib", None)
    monkeypatch.setattr(R, "LIB_PATH", "/nonexistent/libplenreg.so")
    with pytest.raises(R.PlenRegError):
        R.load()


# ---- calls that are recorded or transformed
def _nodes():
    from plen_ml_walk_amd.build import build_regularise, build_regularise_nodes
    build_regularise(), build_regularise_nodes()
    return R._load_nodes()


def recorded_calls(x, call):
    """(kind, the call under it) for every way to record or to transform an operation."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx

    def fake():
        with FakeTensorMode() as mode:
            return call(mode.from_tensor(x))

    yield "trace", lambda: torch.jit.trace(call, x)
    for mode in ("real", "fake", "symbolic"):
        yield "make_fx " + mode, lambda mode=mode: make_fx(call, tracing_mode=mode)(x)
    yield "fake", fake
    yield "vmap", lambda: torch.vmap(call)(x[None].expand(3, *x.shape))
    yield "grad", lambda: torch.func.grad(lambda v: call(v).sum())(x)
    yield "functionalize", lambda: torch.func.functionalize(call)(x)


@pytest.mark.parametrize("kind", ["dropout", "norm", "layer"])
def test_the_nodes_refuse_to_be_recorded(kind):
    """Before anything touches a device, so host tensors will do: what a trace recorded of the kernels' call would be the allocation of its result alone."""
    nodes, x, rng, w = _nodes(), torch.randn(4, 8), R.new_rng("cpu", 1), torch.ones(8)
    call = {"dropout": lambda v: nodes.dropout(v, 100, rng, 0), "norm": lambda v: nodes.norm(v, w, w, 2, 1e-5, 0, 0, None, 0), "layer": lambda v: nodes.norm(v, w, w, 2, 1e-5, 0, 100, rng, 0)}[kind]
    for name, run in recorded_calls(x, call):
        with pytest.raises(RuntimeError, match="plen_ml_walk_amd.regularise"):
            run()


def test_masks_are_not_traced_on_the_cpu():
    x, rng, w = torch.randn(4, 8), R.new_rng("cpu", 1), torch.ones(8)
    for call in (lambda v: R.dropout(v, 0.5, rng), lambda v: R.dropout_norm_act(v, 0.5, rng, 2, w)):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(call, x)
    traced, z = torch.jit.trace(lambda v: R.group_norm_act(v, 2, w), x), torch.randn(4, 8)
    assert torch.equal(traced(z), R.group_norm_act(z, 2, w))
