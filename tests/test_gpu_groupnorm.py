"""ops.group_norm_act (sed_group_norm_fwd / _bwd) against the definition in 64 bits, its gradients against those of the definition and
against differences, and its refusals.

Tolerances count roundings.  H = 2^-24 is half a step of float32.  Outputs of 16 bits add one rounding of their own (eps / 2 of the
type).  In 32 bits the largest terms are: the sums behind mean and variance (chains of at most 64 terms a thread, then trees: 100 H
of the deviation from the group's first values), the mean's own rounding, a few operations, and the activation (12 H of max(1, |z|): exp2 of an argument
rounded at |z| log2(e), a reciprocal, the error function to 1.5e-7 = 2.5 H)."""
import numpy as np
import pytest
import torch

from sound_event_detection_dcase2017_task4_amd import ops

H = 2.0 ** -24
gpu = pytest.mark.gpu
F = torch.nn.functional
ACTS = {"none": lambda z: z, "relu": F.relu, "silu": F.silu, "gelu": F.gelu}
HALF = {torch.float32: 0.0, torch.float16: torch.finfo(torch.float16).eps / 2, torch.bfloat16: torch.finfo(torch.bfloat16).eps / 2}


def _reference(x, w, b, groups, eps, act, gy):
    """y, gx, gw, gb in 64 bits on the CPU, by torch's own autograd."""
    leaf = [t.detach().double().cpu().requires_grad_(True) if t is not None else None for t in (x, w, b)]
    x = leaf[0]
    one = torch.ones(x.shape[-1], dtype=torch.float64)             # torch's own backward wants both parameters or none
    wb = (one if leaf[1] is None else leaf[1], 0 * one if leaf[2] is None else leaf[2])
    z = F.group_norm(x.reshape(x.shape[0], -1, x.shape[-1]).transpose(1, 2), groups, *wb, eps).transpose(1, 2).reshape(x.shape)
    y = ACTS[act](z)
    given = [t for t in leaf if t is not None]
    grads = iter(torch.autograd.grad(y, given, gy.double().cpu()))
    return [y.detach()] + [next(grads) if t is not None else None for t in leaf]


def _inputs(shape, dtype, wdtype, seed, offset=0.5):
    g = torch.Generator().manual_seed(seed)
    C = shape[-1]
    x = torch.randn(shape, generator=g) * (0.5 + torch.rand(C, generator=g)) + offset * torch.randn(C, generator=g)
    w, b = 1 + 0.2 * torch.randn(C, generator=g), 0.2 * torch.randn(C, generator=g)
    gy = torch.randn(shape, generator=g)
    return x.to(dtype).cuda(), w.to(wdtype).cuda(), b.to(wdtype).cuda(), gy.to(dtype).cuda()


def _check(x, w, b, groups, eps, act, gy, offset=0.5):
    """Forward and gradients against 64 bits, elementwise for y, per tensor relative to the largest terms for the gradients."""
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (x, w, b)]
    y = ops.group_norm_act(leaves[0], groups, leaves[1], leaves[2], eps=eps, activation=act)
    assert y.dtype == x.dtype and y.shape == x.shape
    y.backward(gy)
    with torch.no_grad():
        assert torch.equal(ops.group_norm_act(x, groups, w, b, eps=eps, activation=act), y)
    want = _reference(x, w, b, groups, eps, act, gy)
    C, rows = x.shape[-1], x.numel() // (x.shape[0] * x.shape[-1])
    xd = x.double().cpu().reshape(x.shape[0], rows, groups, C // groups)
    rstd = float((1 / torch.sqrt(xd.var(dim=(1, 3), unbiased=False) + eps)).max())
    dev = float((xd - xd[:, :1, :, :1]).abs().max()) * rstd       # largest deviation of a group from one of its members, in units of sigma
    half = HALF[x.dtype]
    wm = float(w.abs().max()) if w is not None else 1.0
    far = float(xd.mean(dim=(1, 3)).abs().max()) * rstd           # the mean itself is a float: off by H of its size
    zerr = (100 + 8 * dev + 2 * far) * H * max(1.0, wm)
    tol_y = half * want[0].abs() * (1 + 2.0 ** -8) + 1.2 * zerr + 12 * H * (1 + want[0].abs()) + (6e-8 if x.dtype == torch.float16 else 0)
    assert ((y.detach().double().cpu() - want[0]).abs() <= tol_y).all(), (y.detach().double().cpu() - want[0]).abs().max()
    # gradients: every term carries zerr through act'' (at most 1.1) and the roundings of its own factors
    gm = float(gy.abs().max()) * 1.2
    terr = (4 * zerr + 40 * H) * gm
    gx = leaves[0].grad.double().cpu()
    big = rstd * wm * (2 + dev)
    assert ((gx - want[1]).abs() <= half * want[1].abs() * (1 + 2.0 ** -8) + 3 * big * terr + (6e-8 if x.dtype == torch.float16 else 0)).all()
    count = x.numel() // C
    for got, ref, scale in ((leaves[1], want[2], 1 + dev), (leaves[2], want[3], 1.0)):
        if got is not None:
            tol = HALF[got.dtype] * ref.abs() * (1 + 2.0 ** -8) + scale * terr * np.sqrt(count) * 4 + (6e-8 if got.dtype == torch.float16 else 0)
            assert got.grad.dtype == got.dtype and ((got.grad.double().cpu() - ref).abs() <= tol).all()


SHAPES = [((1, 1, 8), 2), ((2, 1, 1, 64), 8), ((3, 5, 24), 3), ((2, 33, 51), 17), ((1, 1000, 3), 1), ((2, 777, 7), 7), ((5, 13, 9, 17), 1),
          ((2, 300, 96), 12), ((1, 70, 513), 27), ((2, 9, 2056), 4), ((1, 3, 4100), 5), ((40, 2, 32), 32), ((1, 20011, 40), 5), ((3, 125, 512), 32)]


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape,groups", SHAPES)
def test_against_64_bits(shape, groups, dtype):
    act = list(ACTS)[(len(shape) + shape[1] + shape[-1]) % 4]
    x, w, b, gy = _inputs(shape, dtype, torch.float32, 3)
    if act == "relu":                                    # the mask jumps at 0: keep z away from it
        b = torch.full_like(b, 40.0)
    _check(x, w, b, groups, 1e-3, act, gy)


@gpu
@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_activations_and_parameter_types(act, dtype):
    x, w, b, gy = _inputs((2, 130, 48), dtype, dtype, 5)
    if act == "relu":
        b = torch.where(torch.arange(48, device="cuda") % 2 == 0, 40.0, -40.0).to(dtype)
    _check(x, w, b, 6, 1e-5, act, gy)
    if act != "relu":
        _check(x, None, None, 6, 1e-5, act, gy)
        _check(x, w, None, 6, 1e-5, act, gy)
        _check(x, None, b, 6, 1e-5, act, gy)


@gpu
def test_far_from_zero_and_an_outlier_in_front():
    """Means of a thousand standard deviations, and a first row (the reference point of the sums) far from all others."""
    x, w, b, gy = _inputs((2, 600, 32), torch.float32, torch.float32, 7, offset=0.0)
    x += 1000.0
    # the input itself is rounded at 1000; 64 bits see the same input, so only the kernel's own arithmetic counts
    _check(x, w, b, 4, 1e-5, "silu", gy, offset=0.0)
    x[:, 0] = 0.0
    _check(x, w, b, 4, 1e-5, "silu", gy, offset=0.0)


@gpu
def test_strides_views_and_expanded_gradients():
    x, w, b, gy = _inputs((2, 40, 48), torch.float32, torch.float32, 9)
    ref = ops.group_norm_act(x, 6, w, b, activation="gelu")
    nchw = x.transpose(1, 2).contiguous()                                   # (B, C, rows): channels first in memory
    assert torch.equal(ops.group_norm_act(nchw.transpose(1, 2), 6, w, b, activation="gelu"), ref)
    base = torch.zeros(2 * 40 * 48 + 1, device="cuda")
    base[1:] = x.reshape(-1)
    assert torch.equal(ops.group_norm_act(base[1:].view(2, 40, 48), 6, w, b, activation="gelu"), ref)       # 4-byte aligned only
    assert torch.equal(ops.group_norm_act(x, 6, torch.stack([w, w], 1)[:, 0], b, activation="gelu"), ref)
    leaf = x.clone().requires_grad_(True)
    ops.group_norm_act(leaf, 6, w, b, activation="gelu").sum().backward()  # an expanded gradient
    want = _reference(x, w, b, 6, 1e-5, "gelu", torch.ones_like(x))[1]
    assert (leaf.grad.double().cpu() - want).abs().max() < 2000 * H


@gpu
def test_nan_and_infinity_stay_in_their_group():
    x, w, b, _ = _inputs((3, 50, 32), torch.float32, torch.float32, 11)
    clean = ops.group_norm_act(x, 4, w, b, activation="silu")
    x[1, 20, 9], x[2, 3, 31] = float("nan"), float("inf")
    y = ops.group_norm_act(x, 4, w, b, activation="silu")
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[1, :, 8:16] = bad[2, :, 24:] = True
    assert torch.isnan(y[bad]).all() and torch.equal(y[~bad], clean[~bad])
    z = ops.group_norm_act(torch.full((1, 6, 8), 3.0, device="cuda"), 2, activation="none")   # no variance at all
    assert torch.equal(z, torch.zeros_like(z))


@gpu
def test_empty():
    for shape in ((0, 5, 8), (3, 0, 8)):
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        w = torch.ones(8, device="cuda", requires_grad=True)
        y = ops.group_norm_act(x, 2, w)
        assert y.shape == x.shape
        y.sum().backward()
        assert x.grad.shape == x.shape and not w.grad.any()


@gpu
def test_gradient_against_differences():
    """The loss's change along a direction, by differences of 64-bit references and by the kernel's gradients."""
    x, w, b, gy = _inputs((2, 30, 24), torch.float32, torch.float32, 13)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    (ops.group_norm_act(leaves[0], 3, leaves[1], leaves[2], activation="silu") * gy).sum().backward()
    g = torch.Generator().manual_seed(1)
    for leaf, k in zip(leaves, range(3)):
        d = torch.randn(leaf.shape, generator=g, dtype=torch.float64)
        h = 1e-5
        vals = []
        for s in (h, -h):
            args = [t.detach().double().cpu() for t in (x, w, b)]
            args[k] = args[k] + s * d
            vals.append(float((_reference(*args, 3, 1e-5, "silu", gy)[0] * gy.double().cpu()).sum()))
        slope = (vals[0] - vals[1]) / (2 * h)
        got = float((leaf.grad.double().cpu() * d).sum())
        assert abs(got - slope) < 1e-5 * float(leaf.grad.double().norm()) * float(d.norm()) + 1e-6


@gpu
def test_only_wanted_gradients_and_shared_parameters():
    x, w, b, gy = _inputs((2, 30, 24), torch.float32, torch.float32, 15)
    for k in range(3):
        leaves = [t.clone().requires_grad_(k == j) for j, t in enumerate((x, w, b))]
        ops.group_norm_act(leaves[0], 3, leaves[1], leaves[2], activation="gelu").backward(gy)
        assert [t.grad is not None for t in leaves] == [k == j for j in range(3)]
        want = _reference(x, w, b, 3, 1e-5, "gelu", gy)[1 + k]
        assert (leaves[k].grad.double().cpu() - want).norm() < 1e-5 * want.norm()
    w1 = w.clone().requires_grad_(True)                    # one layer applied twice
    (ops.group_norm_act(x, 3, w1, b) * gy + ops.group_norm_act(2 * x, 3, w1, b) * gy).sum().backward()
    one = w.clone().requires_grad_(True)
    ops.group_norm_act(x, 3, one, b).backward(gy)
    assert (w1.grad - 2 * one.grad).norm() < 1e-4 * one.grad.norm()


@gpu
def test_captured_and_replayed_on_a_side_stream():
    x, w, b, gy = _inputs((4, 200, 64), torch.bfloat16, torch.float32, 17)
    x.requires_grad_(True)
    w.requires_grad_(True)
    run = lambda: torch.autograd.grad(ops.group_norm_act(x, 8, w, b, activation="silu"), (x, w), gy)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for k in range(3):
        with torch.no_grad():
            x.normal_()
            gy.normal_()
        graph.replay()
        torch.cuda.synchronize()
        want = run()
        assert all(torch.equal(a, c) for a, c in zip(got, want)), k


@gpu
def test_more_than_two_to_the_31_elements():
    n, s, c = 3, 2 ** 24 + 5, 48
    x = torch.empty((n, s, c), dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    tile = torch.randn((4099, c), generator=g, device="cuda")
    for k in range(n):                                     # every sample its own scale: a wrong offset shows
        full = ((k + 1) * tile).to(torch.bfloat16)
        x[k, :s // 4099 * 4099] = full.repeat(s // 4099, 1)
        x[k, s // 4099 * 4099:] = full[:s % 4099]
    y = ops.group_norm_act(x, 6)
    for k in range(n):
        part = x[k, :4099].double().view(4099, 6, 8)
        # s = 4092 whole tiles and a rest of 1/4092 of them: the statistics are the tile's to about 1/4092 of sigma
        want = (part - part.mean((0, 2), keepdim=True)) / part.var((0, 2), unbiased=False, keepdim=True).sqrt()
        for at in (0, (s // 4099 - 1) * 4099):
            assert (y[k, at:at + 4099].double().view(4099, 6, 8) - want).abs().max() < 2.0 ** -8 * 6 + 2e-3


@gpu
def test_refusals_on_the_gpu():
    x = torch.zeros(2, 5, 8, device="cuda")
    w = torch.ones(8, device="cuda")
    for args, kw in (((x, 3), {}), ((x, 0), {}), ((x, 2, w[:7]), {}), ((x, 2, w.half()), {}), ((x.double(), 2), {}), ((x[0, 0], 2), {}),
                     ((x, 2, w), {"activation": "tanh"}), ((x, 2, w), {"eps": -1.0}), ((x, 2, w.cpu()), {}), ((x.half(), 2, w, w.half()), {})):
        with pytest.raises(ValueError):
            ops.group_norm_act(*args, **kw)
    x.requires_grad_(True)
    y = ops.group_norm_act(x, 2)
    g, = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_refusals_on_the_cpu():
    x = torch.zeros(2, 5, 8)
    with pytest.raises(RuntimeError):
        ops.group_norm_act(x, 2)
    for bad in (dict(groups=3), dict(groups=2, activation="swish"), dict(groups=2, weight=torch.ones(4)), dict(groups=2, eps=float("nan"))):
        with pytest.raises(ValueError):
            ops.group_norm_act(x, **bad)


def test_c_entries_refuse_bad_arguments():
    from sound_event_detection_dcase2017_task4_amd import _lib
    h = _lib.lib()
    ok = dict(x=1, w=None, b=None, t=0, wt=0, N=2, S=3, C=8, G=2, eps=1e-5, act=0, y=1, m=1, r=1, ws=1)

    def fwd(**kw):
        a = dict(ok, **kw)
        return h.sed_group_norm_fwd(a["x"], a["w"], a["b"], a["t"], a["wt"], a["N"], a["S"], a["C"], a["G"], a["eps"], a["act"], a["y"], a["m"], a["r"], a["ws"], None)

    def bwd(**kw):
        a = dict(ok, **kw)
        return h.sed_group_norm_bwd(a["x"], a["y"], a["w"], a["b"], a["t"], a["wt"], a["N"], a["S"], a["C"], a["G"], a["act"], a["m"], a["r"], None, None, None, a["ws"], None)
    for bad in ({"x": None}, {"y": None}, {"m": None}, {"r": None}, {"t": 3}, {"t": -1}, {"wt": 3}, {"N": 0}, {"S": 0}, {"C": 0}, {"G": 3},
                {"G": 0}, {"act": 4}, {"act": -1}, {"N": 1 << 40}):
        assert fwd(**bad) == -22 and bwd(**bad) == -22, bad
    assert fwd(eps=-1.0) == -22 and fwd(eps=float("nan")) == -22
    assert fwd(S=1 << 20, ws=None) == -22
    assert h.sed_group_norm_ws_floats(0, 2, 3, 8, 3, 0) == 0 and h.sed_group_norm_ws_floats(0, 2, 3, 8, 2, 1) > 0
    assert h.sed_group_norm_ws_floats(0, 2, 1 << 20, 8, 2, 0) > 0


def _large(n, rows, channels, dtype, seed):
    torch.manual_seed(seed)
    x = torch.empty((n, rows, channels), dtype=dtype, device="cuda").normal_()
    x.mul_(torch.linspace(0.5, 2.0, channels, device="cuda").to(dtype)).add_(torch.linspace(-2.0, 3.0, channels, device="cuda").to(dtype))
    return x, 1 + 0.2 * torch.randn(channels, device="cuda"), 0.2 * torch.randn(channels, device="cuda")


LARGE = [(torch.float16, 9, 63337, 384, 8), (torch.bfloat16, 300, 8003, 91, 7), (torch.float32, 64, 16001, 128, 32), (torch.float32, 1030, 100, 1000, 1),
         (torch.float16, 40, 20011, 257, 257)]


@gpu
@pytest.mark.parametrize("dtype,n,rows,channels,groups", LARGE)
def test_samples_shared_by_many_workgroups(dtype, n, rows, channels, groups):
    """Inputs beyond 384 MB: the rows of a sample stay in several workgroups.  Against 64 bits, and bit for bit where they give up at once
    and the second kernel writes the rows, in three launches that follow each other and in two that run side by side."""
    from sound_event_detection_dcase2017_task4_amd import _lib
    x, w, b = _large(n, rows, channels, dtype, 3)
    run = lambda: ops.group_norm_act(x, groups, w, b, activation="silu")  # noqa: E731
    with torch.no_grad():
        y = run()
        for k in {0, n // 2, n - 1}:
            xd = x[k].double().reshape(rows, groups, -1)
            mean, var = xd.mean(dim=(0, 2), keepdim=True), xd.var(dim=(0, 2), keepdim=True, unbiased=False)
            z = ((xd - mean) / torch.sqrt(var + 1e-5)).reshape(rows, channels) * w.double() + b.double()
            want = F.silu(z)
            dev = float((xd - xd[:1]).abs().max() / var.min().sqrt())     # of a channel from its first row
            far = float((mean.abs() / var.sqrt()).max())
            # sums of at most 16 rows a thread, then trees and the joined chunks, as in _check
            zerr = (100 + 8 * dev + 2 * far) * H * float(w.abs().max())
            tol = HALF[dtype] * want.abs() * (1 + 2.0 ** -8) + 1.2 * zerr + 12 * H * (1 + want.abs()) + (6e-8 if dtype == torch.float16 else 0)
            assert ((y[k].double() - want).abs() <= tol).all()
        hooks = _lib.test_hooks()
        try:
            for wait in (1, 0, 1):                         # one tick, the default, one tick
                hooks.sed_gru_set_spin_limit(wait)
                assert torch.equal(run(), y), wait
        finally:
            hooks.sed_gru_set_spin_limit(0)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            a = run()
        c = run()
        torch.cuda.synchronize()
        assert torch.equal(a, y) and torch.equal(c, y)


@gpu
def test_shared_samples_in_a_graph_and_in_training():
    x, w, b = _large(70, 25000, 128, torch.bfloat16, 5)
    with torch.no_grad():
        ops.group_norm_act(x, 8, w, b)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = ops.group_norm_act(x, 8, w, b)
        for _ in range(3):
            x.normal_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, ops.group_norm_act(x, 8, w, b))
    gy = torch.empty_like(x).normal_()
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    got = torch.autograd.grad(ops.group_norm_act(x, 8, w, b, activation="gelu"), leaves, gy)
    part = torch.autograd.grad(ops.group_norm_act(x[:20], 8, w, b, activation="gelu"), leaves, gy[:20])        # 128 MB: in two passes
    # x's gradient: statistics that differ by a few H, then one rounding to bfloat16 each: a step of it apart at most, and mostly equal
    d, s = (got[0][:20].float() - part[0][:20].float()).abs(), part[0][:20].float().abs()
    assert (d <= 2 * HALF[torch.bfloat16] * 1.01 * s + 1e-5 * s.max()).all() and (d > 0).float().mean() < 0.01


@gpu
def test_a_nan_and_an_infinity_stay_in_their_sample_when_shared():
    x, w, b = _large(70, 25000, 128, torch.bfloat16, 6)
    with torch.no_grad():
        clean = ops.group_norm_act(x, 8, w, b, activation="relu")
        x[3, 24999, 5], x[40, 0, 127] = float("nan"), float("inf")
        y = ops.group_norm_act(x, 8, w, b, activation="relu")
    bad = torch.zeros(70, 8, dtype=torch.bool, device="cuda")
    bad[3, 0], bad[40, 7] = True, True
    nan = torch.isnan(y).reshape(70, 25000, 8, 16)
    assert torch.equal(nan.all(dim=3).all(dim=1), bad) and torch.equal(nan.any(dim=3).any(dim=1), bad)
    keep = ~bad.view(70, 1, 8, 1).expand(70, 25000, 8, 16).reshape(y.shape)
    assert torch.equal(y[keep], clean[keep])


def test_c_entries_refuse_what_a_launch_cannot_hold():
    from sound_event_detection_dcase2017_task4_amd import _lib
    h = _lib.lib()
    for t in (0, 1, 2):
        for n, s, c, g in ((1 << 22, 1, 8, 1), (1 << 14, 1, 256, 256), (1 << 21, 1 << 20, 64, 1), (1 << 11, 1, 1 << 22, 1)):
            assert h.sed_group_norm_ws_floats(t, n, s, c, g, 1) == 0
            assert h.sed_group_norm_fwd(16, None, None, t, 0, n, s, c, g, 1e-5, 0, 16, 16, 16, 16, None) == -22
            assert h.sed_group_norm_bwd(16, 16, None, None, t, 0, n, s, c, g, 0, 16, 16, None, None, None, 16, None) == -22


@gpu
@pytest.mark.parametrize("shape,groups", [((3, 300, 64), 4), ((2, 1000, 24), 3), ((2, 9000, 40), 5), ((1, 40000, 16), 2), ((7, 8, 8), 1), ((6, 125000, 256), 8)])
@pytest.mark.parametrize("where", [0, -1, 17])
def test_a_row_far_from_the_others(shape, groups, where):
    """One row of zeros (a padded frame) beside rows around 1000 sigma: the variance is that row's, but for its sixteenth digit the rest's.
    A thread reads at most 64 rows of a channel, and sums squares of distances from the first of them: 64 D^2, each product and sum
    rounded (3 H), against the D^2 that the row adds to the group -- 200 H of the variance at most, half of that of 1 / sigma; the mean is rounded
    for a thread, a workgroup, a group and a sample, and is off by 6 H of itself at most, which is up to sqrt(rows) sigma."""
    g = torch.Generator(device="cuda").manual_seed(7)
    x = 1000.0 + torch.randn(shape, generator=g, device="cuda")
    x[:, where % shape[1]] = 0.0
    with torch.no_grad():
        y = ops.group_norm_act(x, groups)
    xd = x.double().reshape(shape[0], shape[1], groups, -1)
    mean, var = xd.mean(dim=(1, 3), keepdim=True), xd.var(dim=(1, 3), keepdim=True, unbiased=False)
    want = ((xd - mean) / torch.sqrt(var + 1e-5)).reshape(shape)
    far = float((mean.abs() / var.sqrt()).max())
    assert ((y.double() - want).abs() <= 100 * H * want.abs() + 6 * H * far + 4 * H).all()


@gpu
@pytest.mark.parametrize("shape,groups", [((2, 130, 48), 6), ((2, 9000, 40), 5)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_relu_selects_its_gradient(shape, groups, dtype):
    """As torch: an infinite gradient does not come through a unit that is off, and a unit whose z is NaN is on (in one pass and in two)."""
    C = shape[-1]
    x, w, b, gy = _inputs(shape, dtype, torch.float32, 19)
    b = torch.where(torch.arange(C, device="cuda") % 2 == 0, 40.0, -40.0)
    b[9] = float("nan")                                      # a bias enters no sum but its own channel's
    gy[0, 3, 1], gy[1, 7, 5] = float("inf"), float("nan")
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    got = torch.autograd.grad(ops.group_norm_act(leaves[0], groups, leaves[1], leaves[2], activation="relu"), leaves, gy)
    want = _reference(x, w, b, groups, 1e-5, "relu", gy)[1:]
    assert all(torch.isfinite(t).all() for t in want)
    for a, c in zip(got, want):
        # normwise: sums of about a hundred H (as in _check) beside the output's own rounding
        assert float((a.double().cpu() - c).norm()) <= (200 * H + HALF[a.dtype]) * float(c.norm())


def test_c_entries_refuse_more_channels_than_the_parameter_sums_hold():
    from sound_event_detection_dcase2017_task4_amd import _lib
    h = _lib.lib()
    for t in (0, 1, 2):
        for n, s, c, g in ((1, 1, 1 << 26, 1 << 20), (1, 1, 1 << 26, 1 << 21), (1, 3, (1 << 26) + 4096, 1 << 12)):
            for backward in (0, 1):
                assert h.sed_group_norm_ws_floats(t, n, s, c, g, backward) == 0
            assert h.sed_group_norm_fwd(16, None, None, t, 0, n, s, c, g, 1e-5, 0, 16, 16, 16, 16, None) == -22
            assert h.sed_group_norm_bwd(16, 16, None, None, t, 0, n, s, c, g, 0, 16, 16, None, 16, 16, 16, None) == -22


@gpu
@pytest.mark.parametrize("shape,groups", [((2, 9000, 40), 5), ((3, 40001, 24), 3), ((2, 6001, 51), 17)])
def test_only_wanted_gradients_in_two_passes(shape, groups):
    """Rows that a workgroup cannot hold: the parameters' sums have a launch of their own where x needs no gradient.  They are the sums of the
    same numbers as beside gx, added in another order: a hundred H of them in the norm, as in _check."""
    x, w, b, gy = _inputs(shape, torch.float32, torch.float32, 15)
    full = [t.clone().requires_grad_(True) for t in (x, w, b)]
    every = torch.autograd.grad(ops.group_norm_act(full[0], groups, full[1], full[2], activation="gelu"), full, gy)
    want = _reference(x, w, b, groups, 1e-5, "gelu", gy)[1:]
    for wanted in ((0,), (1,), (2,), (1, 2), (0, 2)):
        leaves = [t.clone().requires_grad_(j in wanted) for j, t in enumerate((x, w, b))]
        got = torch.autograd.grad(ops.group_norm_act(leaves[0], groups, leaves[1], leaves[2], activation="gelu"), [leaves[j] for j in wanted], gy)
        for j, t in zip(wanted, got):
            assert float((t.double().cpu() - want[j]).norm()) <= 200 * H * float(want[j].norm()) and float((t - every[j]).norm()) <= 100 * H * float(every[j].norm())
