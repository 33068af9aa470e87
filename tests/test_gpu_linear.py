"""ops.linear_act (sed_linear_fwd / _bwd) against the definition in 64 bits, its gradients, and its refusals.

Tolerances count roundings.  H = 2^-24 is half a step of float32, e = eps / 2 of a 16-bit type (0 for float32).  A sum of K products
in 32 bits is off by at most K H of the sum of their magnitudes; the bound used is half of that with a floor for short sums, as the
roundings of a chain do not all point one way.  An output adds one rounding e of itself.  In the backward pass gz carries one rounding
e (for the two products) and, behind an activation, the rounding of the kept z to float16 (2^-11 of z; |act''| <= 1.2)."""
import math

import pytest
import torch

from sound_event_detection_dcase2017_task4_amd import ops

H = 2.0 ** -24
gpu = pytest.mark.gpu
F = torch.nn.functional
ACTS = {"none": lambda z: z, "relu": F.relu, "silu": F.silu, "gelu": F.gelu}
HALF = {torch.float32: 0.0, torch.float16: torch.finfo(torch.float16).eps / 2, torch.bfloat16: torch.finfo(torch.bfloat16).eps / 2}
TINY = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}         # half a step of float16's smallest numbers
TYPES = list(HALF)


def _inputs(m, k, n, dtype, btype, seed, residual=True):
    g = torch.Generator().manual_seed(seed)
    x, w, b = torch.randn(m, k, generator=g), torch.randn(n, k, generator=g) / math.sqrt(k), 0.2 * torch.randn(n, generator=g)
    r, gy = torch.randn(m, n, generator=g), torch.randn(m, n, generator=g)
    return x.to(dtype).cuda(), w.to(dtype).cuda(), b.to(btype).cuda(), r.to(dtype).cuda() if residual else None, gy.to(dtype).cuda()


def _sum_err(count):
    return (0.5 * count + 16) * H


def _check(x, w, b, r, gy, act):
    leaves = [t.detach().clone().requires_grad_(True) if t is not None else None for t in (x, w, b, r)]
    y = ops.linear_act(leaves[0], leaves[1], leaves[2], activation=act, residual=leaves[3])
    y.backward(gy)
    with torch.no_grad():
        assert torch.equal(ops.linear_act(x, w, b, activation=act, residual=r), y)
    d = lambda t: None if t is None else t.detach().double()  # noqa: E731
    xd, wd, bd, rd, gd = d(x), d(w), d(b), d(r), d(gy)
    (M, K), N = x.shape, w.shape[0]
    e, tiny = HALF[x.dtype], TINY[x.dtype]
    z = (xd @ wd.t() + (0 if bd is None else bd)).requires_grad_(True)
    a = ACTS[act](z)
    da, = torch.autograd.grad(a.sum(), z)
    z, a = z.detach(), a.detach()
    want = a + (0 if rd is None else rd)
    zerr = _sum_err(K) * (xd.abs() @ wd.abs().t() + (0 if bd is None else bd.abs())) + 4 * H
    tol = 1.2 * zerr + 12 * H * (1 + want.abs()) + e * 1.01 * want.abs() + tiny
    assert y.dtype == x.dtype and ((y.detach().double() - want).abs() <= tol).all()
    gz = gd * da
    kept = (2.0 ** -11 * z.abs() + 2.0 ** -25 if x.dtype != torch.float32 else 0) if act in ("silu", "gelu") else 0
    gzerr = gd.abs() * (1.2 * (kept + zerr) + 16 * H) + e * 1.01 * gz.abs() + tiny
    gx, gw = gz @ wd, gz.t() @ xd
    tx = gzerr @ wd.abs() + _sum_err(N) * (gz.abs() @ wd.abs()) + e * 1.01 * gx.abs() + tiny
    tw = gzerr.t() @ xd.abs() + _sum_err(M) * (gz.abs().t() @ xd.abs()) + e * 1.01 * gw.abs() + tiny
    assert ((leaves[0].grad.double() - gx).abs() <= tx).all() and ((leaves[1].grad.double() - gw).abs() <= tw).all()
    assert leaves[0].grad.dtype == x.dtype and leaves[1].grad.dtype == w.dtype
    if b is not None:
        eb = HALF[b.dtype]
        tb = (gd.abs() * (1.2 * (kept + zerr) + 16 * H)).sum(0) + _sum_err(M) * gz.abs().sum(0) + eb * 1.01 * gz.sum(0).abs() + TINY[b.dtype]
        assert leaves[2].grad.dtype == b.dtype and ((leaves[2].grad.double() - gz.sum(0)).abs() <= tb).all()
    if r is not None:
        assert torch.equal(leaves[3].grad, gy)


SHAPES = [(1, 1, 1), (1, 512, 2048), (2, 7, 5), (15, 64, 16), (16, 200, 33), (17, 65, 130), (64, 513, 48), (65, 8, 8), (65, 9, 7), (128, 128, 128),
          (129, 72, 257), (200, 1000, 17), (127, 63, 255), (1001, 513, 127), (300, 40, 1000), (513, 256, 512), (2000, 96, 24), (5, 3000, 12)]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_against_64_bits(m, k, n, dtype):
    # LDS and scratch hold NaN when the case begins: what is read beside the matrix shows
    bad = torch.full((300, 300), float("nan"), dtype=dtype, device="cuda")
    ops.linear_act(bad, bad)
    act = ("none", "silu", "gelu")[(m + k + n) % 3]
    _check(*_inputs(m, k, n, dtype, dtype, m + k, residual=(m + n) % 2 == 0), act)


@gpu
@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("dtype", TYPES)
def test_activations_biases_and_residuals(act, dtype):
    for m in (3, 150):
        x, w, b, r, gy = _inputs(m, 96, 40, dtype, torch.float32, 7)
        if act == "relu":                                  # the mask jumps at 0: keep z away from it, on both sides
            b = torch.where(torch.arange(40, device="cuda") % 2 == 0, 30.0, -30.0)
        _check(x, w, b, r, gy, act)
        _check(x, w, b, None, gy, act)
        if act != "relu":
            _check(x, w, None, r, gy, act)
            _check(x, w, b.to(dtype), r, gy, act)


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_pre_activations_beyond_the_kept_range(dtype):
    """|z| beyond 60000 is kept clamped: the derivative is 1 or 0 there all the same.  ReLU keeps its mask for the smallest z."""
    x = torch.full((70, 8), 180.0, dtype=dtype, device="cuda")
    w = torch.tensor([100.0] * 8 + [-100.0] * 8, device="cuda").view(2, 8).to(dtype).requires_grad_(True)
    for act in ("silu", "gelu"):
        y = ops.linear_act(x.float(), w.float(), activation=act)       # 144000 fits float32 and bfloat16
        g, = torch.autograd.grad(y.sum(), w)
        assert torch.equal(g, torch.tensor([[12600.0] * 8, [0.0] * 8], device="cuda").to(dtype))
    if dtype == torch.bfloat16:
        for act in ("silu", "gelu", "relu"):
            g, = torch.autograd.grad(ops.linear_act(x, w, activation=act).sum(), w)
            assert torch.equal(g, torch.tensor([[12600.0] * 8, [0.0] * 8], device="cuda").to(dtype))
    small = torch.full((70, 8), 2.0 ** -14, dtype=dtype, device="cuda")
    v = torch.full((2, 8), 2.0 ** -14, dtype=dtype, device="cuda").requires_grad_(True)
    g, = torch.autograd.grad(ops.linear_act(small, v, activation="relu").sum(), v)       # z = 2^-25
    assert torch.equal(g, torch.full_like(v, 70 * 2.0 ** -14))


@gpu
def test_nan_and_infinity_reach_only_their_rows():
    for m in (6, 200):
        x, w, b, _, _ = _inputs(m, 72, 130, torch.bfloat16, torch.float32, 3)
        clean = ops.linear_act(x, w, b, activation="gelu")
        x[2, 5], x[4, 71] = float("nan"), float("inf")
        y = ops.linear_act(x, w, b, activation="gelu")
        ok = torch.ones(m, dtype=torch.bool, device="cuda")
        ok[2] = ok[4] = False
        assert torch.equal(y[ok], clean[ok]) and torch.isnan(y[2]).all() and not torch.isfinite(y[4]).all()


@gpu
def test_strides_views_and_leading_dimensions():
    x, w, b, r, gy = _inputs(120, 64, 48, torch.float16, torch.float16, 5)
    ref = ops.linear_act(x, w, b, "silu", r)
    x3, r3 = x.view(4, 30, 64), r.view(4, 30, 48)
    assert torch.equal(ops.linear_act(x3, w, b, "silu", r3), ref.view(4, 30, 48))
    assert torch.equal(ops.linear_act(x3.transpose(0, 1), w, b, "silu", r3.transpose(0, 1)), ref.view(4, 30, 48).transpose(0, 1))
    assert torch.equal(ops.linear_act(x, w.t().contiguous().t(), b, "silu", r), ref)
    for shift in (1, 2, 4):                                  # 2-, 4- and 8-byte aligned operands
        def moved(t):
            base = torch.zeros(t.numel() + 8, dtype=t.dtype, device="cuda")
            base[shift:shift + t.numel()] = t.reshape(-1)
            return base[shift:shift + t.numel()].view(t.shape)
        assert torch.equal(ops.linear_act(moved(x), moved(w), moved(b), "silu", moved(r)), ref)
        assert torch.equal(ops.linear_act(moved(x)[:7], moved(w), moved(b), "silu", moved(r)[:7]), ops.linear_act(x[:7], w, b, "silu", r[:7]))
        grads = []
        for f in (torch.clone, moved):
            leaves = [f(t).requires_grad_(True) for t in (x, w, b)]
            grads.append(torch.autograd.grad(ops.linear_act(*leaves, "silu"), leaves, f(gy)))
        assert all(torch.equal(p, q) for p, q in zip(*grads))
    one = ops.linear_act(x[0], w, b, "silu")                 # a single vector
    assert one.shape == (48,) and torch.equal(one, ops.linear_act(x[:1], w, b, "silu")[0])
    leaf = x.clone().requires_grad_(True)
    ops.linear_act(leaf, w).sum().backward()                 # an expanded gradient
    want = w.double().sum(0)
    assert ((leaf.grad.double() - want).abs() <= 2.0 ** -11 * want.abs() + _sum_err(48) * w.double().abs().sum(0)).all()


@gpu
def test_empty_and_only_wanted_gradients():
    w = torch.ones(5, 8, device="cuda", requires_grad=True)
    for shape in ((0, 8), (3, 0, 8)):
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        y = ops.linear_act(x, w, activation="gelu")
        assert y.shape == shape[:-1] + (5,)
        y.sum().backward()
        assert x.grad.shape == x.shape and not w.grad.any()
    x, w, b, r, gy = _inputs(100, 40, 24, torch.float32, torch.float32, 9)
    full = [t.clone().requires_grad_(True) for t in (x, w, b, r)]
    want = torch.autograd.grad(ops.linear_act(full[0], full[1], full[2], "silu", full[3]), full, gy)
    for k in range(4):
        leaves = [t.clone().requires_grad_(k == j) for j, t in enumerate((x, w, b, r))]
        got, = torch.autograd.grad(ops.linear_act(leaves[0], leaves[1], leaves[2], "silu", leaves[3]), [leaves[k]], gy)
        assert torch.equal(got, want[k])
    shared = w.clone().requires_grad_(True)                  # one weight used twice
    (ops.linear_act(x, shared) + ops.linear_act(x, shared)).backward(gy)
    once, = torch.autograd.grad(ops.linear_act(x, full[1]), [full[1]], gy)
    assert (shared.grad - 2 * once).norm() < 1e-5 * once.norm()


@gpu
def test_gradient_against_differences():
    x, w, b, r, gy = _inputs(90, 40, 24, torch.float32, torch.float32, 13)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    (ops.linear_act(leaves[0], leaves[1], leaves[2], "gelu", r) * gy).sum().backward()
    g = torch.Generator().manual_seed(1)
    for k, leaf in enumerate(leaves):
        d = torch.randn(leaf.shape, generator=g, dtype=torch.float64).cuda()
        vals = []
        for s in (1e-5, -1e-5):
            args = [t.double() for t in (x, w, b)]
            args[k] = args[k] + s * d
            vals.append(float((F.gelu(args[0] @ args[1].t() + args[2]) * gy.double()).sum()))
        got = float((leaf.grad.double() * d).sum())
        assert abs(got - (vals[0] - vals[1]) / 2e-5) < 1e-5 * float(leaf.grad.double().norm()) * float(d.norm())


@gpu
def test_long_contraction_is_cut_and_repeats_bit_for_bit():
    x, w, b, _, gy = _inputs(20000, 64, 48, torch.bfloat16, torch.float32, 17, residual=False)
    _check(x, w, b, None, gy, "silu")
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    first = torch.autograd.grad(ops.linear_act(*leaves, "silu"), leaves, gy)
    for _ in range(3):
        again = torch.autograd.grad(ops.linear_act(*leaves, "silu"), leaves, gy)
        assert all(torch.equal(p, q) for p, q in zip(first, again))


@gpu
def test_captured_replayed_and_two_graphs_side_by_side():
    x, w, b, r, gy = _inputs(300, 136, 72, torch.bfloat16, torch.float32, 19)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    run = lambda: torch.autograd.grad(ops.linear_act(x, w, b, "gelu", r), leaves, gy)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            run()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(run())
    for k in range(3):
        with torch.no_grad():
            x.normal_()
            gy.normal_()
        side.wait_stream(torch.cuda.current_stream())
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        torch.cuda.synchronize()
        want = run()
        for got in outs:
            assert all(torch.equal(p, q) for p, q in zip(got, want)), k


@gpu
def test_more_than_two_to_the_31_elements():
    M, K, N = 2 ** 25 + 130, 72, 40
    x = torch.zeros((M, K), dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    tail = torch.randn((300, K), generator=g, device="cuda").to(torch.bfloat16)
    w = torch.randn((N, K), generator=g, device="cuda").to(torch.bfloat16).requires_grad_(True)
    x[-300:] = tail
    y = ops.linear_act(x, w)
    assert torch.equal(y[-300:].detach(), ops.linear_act(tail, w.detach())) and not y[:100000].any()
    gy = torch.zeros_like(y)
    gy[-300:] = torch.randn((300, N), generator=g, device="cuda").to(torch.bfloat16)
    gw, = torch.autograd.grad(y, [w], gy)
    want = gy[-300:].double().t() @ tail.double()
    # bfloat16 keeps 8 bits, the first of them fixed: its numbers lie 2^-7 apart relative to the power of two below, half of that is 2^-8
    assert ((gw.double() - want).abs() <= HALF[torch.bfloat16] * 1.01 * want.abs() + _sum_err(300) * (gy[-300:].double().abs().t() @ tail.double().abs())).all()


@gpu
def test_refusals_on_the_gpu():
    x, w, b, r, _ = _inputs(6, 8, 4, torch.float32, torch.float32, 1)
    for args in ((x, w[:, :7]), (x, w.half()), (x.double(), w.double()), (x, w, b[:3]), (x, w, b.half()), (x, w, b, "tanh"), (x, w, b, "none", r[:5]),
                 (x, w, b, "none", r.half()), (x, w.cpu()), (x, w[0]), (x[:, :0], w[:, :0]), (x, w[:0])):
        with pytest.raises(ValueError):
            ops.linear_act(*args)
    x.requires_grad_(True)
    g, = torch.autograd.grad(ops.linear_act(x, w, b, "silu").sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_refusals_on_the_cpu():
    x, w = torch.zeros(3, 8), torch.zeros(4, 8)
    with pytest.raises(RuntimeError):
        ops.linear_act(x, w)
    for args in ((x, w[:, :5]), (x, w.half()), (x, w, torch.zeros(5)), (x, w, None, "tanh"), (x, w, None, "none", torch.zeros(3, 5))):
        with pytest.raises(ValueError):
            ops.linear_act(*args)


def test_c_entries_refuse_bad_arguments():
    from sound_event_detection_dcase2017_task4_amd import _lib
    h = _lib.lib()
    ok = dict(x=16, w=16, t=1, bt=1, M=100, N=8, K=8, act=0, y=16, z=None, ws=None, n=0, gy=16, gx=16, gw=None, gb=None)

    def fwd(**kw):
        a = dict(ok, **kw)
        return h.sed_linear_fwd(a["x"], a["w"], None, None, a["t"], a["bt"], a["M"], a["N"], a["K"], a["act"], a["y"], a["z"], a["ws"], a["n"], None)

    def bwd(**kw):
        a = dict(ok, **kw)
        return h.sed_linear_bwd(a["x"], a["w"], a["gy"], a["z"], a["t"], a["bt"], a["M"], a["N"], a["K"], a["act"], a["gx"], a["gw"], a["gb"], a["ws"], a["n"], None)
    common = ({"t": 3}, {"t": -1}, {"bt": 3}, {"M": 0}, {"N": 0}, {"K": 0}, {"act": 4}, {"N": 1 << 22}, {"K": 1 << 22}, {"M": 1 << 31}, {"w": None},
              {"K": 9}, {"K": 9, "ws": 16, "n": 64})                     # a K that needs scratch, without it or with too little
    for bad in common + ({"x": None}, {"y": None}):
        assert fwd(**bad) == -22, bad
    for bad in common + ({"gy": None}, {"act": 2}, {"gw": 16, "x": None}, {"N": 9}, {"gb": 16}):
        assert bwd(**bad) == -22, bad
    assert h.sed_linear_fwd_ws_bytes(16, 16, 1, 100, 8, 9) > 0 and h.sed_linear_fwd_ws_bytes(16, 16, 1, 64, 8, 9) == 0
    assert h.sed_linear_fwd_ws_bytes(16, 16, 1, 0, 8, 9) == 0 and h.sed_linear_kept_elements(3, 9) == 48


def test_c_entries_refuse_what_a_launch_cannot_hold():
    from sound_event_detection_dcase2017_task4_amd import _lib
    h = _lib.lib()
    for t in (0, 1, 2):
        for m, n, k in ((1 << 30, 4096, 8), (1 << 30, 8, 4096), (1 << 21, 1 << 21, 8), (8, 1 << 21, 1 << 21), ((1 << 31) - 256, 8, 8)):
            assert h.sed_linear_fwd_ws_bytes(16, 16, t, m, n, k) == 0
            assert h.sed_linear_fwd(16, 16, None, None, t, t, m, n, k, 0, 16, None, 16, 1 << 60, None) == -22
            assert h.sed_linear_bwd(16, 16, 16, None, t, t, m, n, k, 0, 16, None, None, 16, 1 << 60, None) == -22


@gpu
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [1, 5, 70, 700])
def test_bias_gradient_of_16_bit_tensors_has_the_bits_of_its_own_type(m, dtype, act):
    """A 32-bit bias beside 16-bit tensors: the derivative is that of z in 32 bits, so the roundings of the tensors' type do not enter."""
    x, w, b, _, gy = _inputs(m, 96, 40, dtype, torch.float32, 31, residual=False)
    b.requires_grad_(True)
    got, = torch.autograd.grad(ops.linear_act(x, w, b, act), b, gy)
    xd, wd, gd = x.double(), w.double(), gy.double()
    z = (xd @ wd.t() + b.detach().double()).requires_grad_(True)
    da, = torch.autograd.grad(ACTS[act](z).sum(), z)
    zerr = _sum_err(96) * (xd.abs() @ wd.abs().t() + b.detach().double().abs()) + 4 * H
    tol = (gd.abs() * (1.2 * zerr + 16 * H)).sum(0) + _sum_err(m) * (gd * da).abs().sum(0)
    assert got.dtype == torch.float32 and ((got.double() - (gd * da).sum(0)).abs() <= tol).all()


def _gradients(x, w, gy, act):
    """gx and gw of linear_act, those of the formula in 64 bits, and gz."""
    leaves = [t.clone().requires_grad_(True) for t in (x, w)]
    got = torch.autograd.grad(ops.linear_act(*leaves, activation=act), leaves, gy)
    z = (x.double() @ w.double().t()).requires_grad_(True)
    gz = gy.double() * torch.autograd.grad(ACTS[act](z).sum(), z)[0]
    return got, (gz @ w.double(), gz.t() @ x.double()), gz


PARTS = [(70, 40, 24), (64, 128, 64), (129, 72, 257), (300, 136, 65), (1001, 520, 127), (4000, 512, 200), (20000, 64, 48), (65, 9, 7), (3, 200, 33)]


@gpu
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,k,n", PARTS)
def test_gradients_of_16_bit_tensors_carry_one_rounding(m, k, n, dtype, act):
    """gz enters the products as the sum of two numbers of the type: off by e^2 of itself (float16: and 2^-36), e half a step of the type.  What
    is left beside the sums' roundings is the gradient's own."""
    x, w, _, _, gy = _inputs(m, k, n, dtype, dtype, 37, residual=False)
    e, tiny = HALF[dtype], TINY[dtype]
    for scale in (1.0, 2.0 ** -18):                         # the second one: a large share of the gradient is below float16's normal numbers
        g = (gy.float() * scale).to(dtype)
        got, want, gz = _gradients(x, w, g, act)
        zerr = _sum_err(k) * (x.double().abs() @ w.double().abs().t()) + 4 * H
        gzerr = g.double().abs() * (1.2 * zerr + 16 * H) + e * e * gz.abs() + (2.0 ** -36 if dtype == torch.float16 else 0)
        for a, b, err, terms in ((got[0], want[0], gzerr @ w.double().abs(), _sum_err(2 * n) * (gz.abs() @ w.double().abs())),
                                 (got[1], want[1], gzerr.t() @ x.double().abs(), _sum_err(2 * m) * (gz.abs().t() @ x.double().abs()))):
            assert ((a.double() - b).abs() <= err + terms + e * 1.01 * b.abs() + tiny).all()
            # and in the norm: within a twentieth of what rounding the right gradient leaves
            assert (a.double() - b).norm() <= 1.05 * (b.to(dtype).double() - b).norm()


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_gradients_at_the_ends_of_the_range(dtype):
    x, w, _, _, gy = _inputs(150, 64, 96, dtype, dtype, 41, residual=False)
    gy = torch.zeros_like(gy)
    x[5], w[7] = 2.0 ** -6, 1.5                             # z = 1.5, where GELU's derivative is 1.13: gz is beyond float16's largest number
    gy[5, 7] = 60000.0
    got, want, gz = _gradients(x, w, gy, "gelu")
    assert float(gz[5, 7]) > 65504
    assert torch.equal(got[1], want[1].to(dtype)) and torch.equal(got[0][:5], torch.zeros_like(got[0][:5]))
    for bad in (float("inf"), -float("inf"), float("nan")):
        x, w, _, _, gy = _inputs(150, 64, 96, dtype, dtype, 43, residual=False)
        clean = _gradients(x, w, gy, "silu")[0]
        gy[5, 7] = bad
        got, want, _ = _gradients(x, w, gy, "silu")
        for a, b, c, at in ((got[0], want[0], clean[0], 5), (got[1], want[1], clean[1], 7)):
            keep = torch.arange(len(a), device="cuda") != at
            assert torch.equal(a[keep], c[keep]) and not torch.isfinite(a[at]).any()
            assert torch.equal(a[at].double().nan_to_num(1.0, 2.0, 3.0), b[at].nan_to_num(1.0, 2.0, 3.0))


@gpu
@pytest.mark.parametrize("m", [50, 200001])
def test_gelu_and_its_derivative_over_the_range(m):
    """z Phi(z) with Phi(-|z|) right to a few roundings of itself: 16 H for the polynomial, the reciprocal and the products, and 1.5 z^2 H for
    the exponential's argument z^2 / 2, which is rounded three times.  A positive z takes them of 1 - Phi and adds two of its own.  The
    derivative has the same in Phi and in z phi."""
    z = torch.linspace(-9.0, 9.0, m, device="cuda").view(-1, 1).requires_grad_(True)
    one = torch.ones(1, 1, device="cuda")
    y = ops.linear_act(z, one, activation="gelu")
    g, = torch.autograd.grad(y.sum(), z)
    zd = z.detach().double()
    tail, phi = 0.5 * torch.erfc(zd.abs() / 2 ** 0.5), torch.exp(-0.5 * zd * zd) / math.sqrt(2 * math.pi)
    cdf = torch.where(zd < 0, tail, 1 - tail)
    near = (16 + 1.5 * zd * zd) * H
    terr = tail * near + torch.where(zd < 0, 0.0, 2 * H)
    assert ((y.detach().double() - zd * cdf).abs() <= zd.abs() * terr + 2.0 ** -126).all()
    assert ((g.double() - (cdf + zd * phi)).abs() <= terr + zd.abs() * phi * near + 2 * H * (cdf + zd * phi).abs() + 2.0 ** -126).all()


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [6, 200])
def test_relu_passes_the_gradient_of_a_nan(m, dtype):
    """As torch: a unit whose z is NaN is on, and a gradient that is not finite does not come through one that is off."""
    x, w, b, _, gy = _inputs(m, 40, 24, dtype, dtype, 51, residual=False)
    b = torch.where(torch.arange(24, device="cuda") % 2 == 0, 30.0, -30.0).to(dtype)
    b[3], gy[2, 5] = float("nan"), float("inf")              # unit 5 is off
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    got = torch.autograd.grad(ops.linear_act(*leaves, activation="relu"), leaves, gy)
    d = [t.detach().double().requires_grad_(True) for t in (x, w, b)]
    want = torch.autograd.grad(F.relu(F.linear(*d)), d, gy.double())
    on = (torch.arange(24, device="cuda") % 2 == 0) | (torch.arange(24, device="cuda") == 3)
    gz = torch.where(on, gy.double(), 0.0)
    terms = (_sum_err(24) * (gz.abs() @ d[1].abs()), _sum_err(m) * (gz.abs().t() @ d[0].abs()), _sum_err(m) * gz.abs().sum(0))
    for a, c, t in zip(got, want, terms):
        assert ((a.double() - c).abs() <= t.detach() + HALF[dtype] * 1.01 * c.abs() + TINY[dtype]).all()
    w[3, 7] = float("nan")                                   # a NaN that comes in through W: rows of gx are NaN there and nowhere else
    leaves[1] = w.clone().requires_grad_(True)
    leaves[2] = torch.where(torch.isnan(b), torch.zeros_like(b), b).requires_grad_(True)
    got = torch.autograd.grad(ops.linear_act(*leaves, activation="relu"), leaves, gy)
    d = [t.detach().double().requires_grad_(True) for t in leaves]
    want = torch.autograd.grad(F.relu(F.linear(*d)), d, gy.double())
    assert all(torch.equal(torch.isnan(a), torch.isnan(c)) for a, c in zip(got, want))


# Shapes whose products are cut into tiles of 128 and 256: (which product, edge, cut along k), rows, K, N.  No size is a multiple of 64, so that
# every one ends inside a tile and inside a step; the second shape of each pair has lines that are not aligned.
WIDE16 = [(0, 128, False, 33772, 40, 72), (0, 128, False, 37109, 40, 67), (0, 128, True, 67, 5224, 4312), (0, 128, True, 3074, 5501, 65),
          (0, 256, False, 26822, 1064, 408), (0, 256, False, 19870, 1033, 540)]
BACK16 = [(1, 128, False, 33035, 72, 40), (1, 128, False, 33885, 68, 46), (1, 128, True, 73, 3384, 5968), (1, 128, True, 4297, 66, 4609),
          (1, 256, False, 25665, 400, 1104), (1, 256, False, 19738, 522, 1061), (2, 128, False, 65, 880, 4704), (2, 128, False, 66, 3590, 1115),
          (2, 128, True, 4365, 4248, 72), (2, 128, True, 5554, 3077, 65), (2, 256, False, 1050, 3352, 3656), (2, 256, False, 1031, 3245, 3836),
          (2, 256, True, 38925, 392, 3144), (2, 256, True, 38748, 3106, 386)]
WIDE32 = [(0, 28623, 40, 144), (0, 21371, 42, 206), (0, 66, 2072, 4640), (0, 4153, 2061, 66), (1, 28303, 144, 40), (1, 27290, 130, 49),
          (1, 4294, 80, 2120), (1, 67, 4227, 2093), (2, 67, 4904, 1080), (2, 67, 2638, 1933), (2, 2218, 80, 4272), (2, 2227, 4119, 66)]


def _plan(dtype, m, k, n, act, which):
    """(edge, slices) of one product of a call."""
    from sound_event_detection_dcase2017_task4_amd import _lib
    p = _lib.lib().sed_linear_plan(ops.DTYPE_CODES[dtype], m, n, k, ops.ACTIVATIONS[act], which)
    return p % 1024, p // 1024


def _poison(dtype):
    """LDS and scratch hold NaN when the case begins: what is read beside the matrices shows."""
    ops.linear_act(*[torch.full((4000, 1000), float("nan"), dtype=dtype, device="cuda")] * 2)


@gpu
@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("which,edge,cut,m,k,n", WIDE16)
def test_forward_in_larger_tiles(which, edge, cut, m, k, n, dtype, act):
    got = _plan(dtype, m, k, n, act, which)
    assert got[0] == edge and (got[1] > 1) == cut
    x, w, b, r, _ = _inputs(m, k, n, dtype, dtype, 61)
    _poison(dtype)
    for bias, res in ((b, r), (b.float(), None), (None, r)):
        leaf = x.clone().requires_grad_(True)              # z is kept, or its mask
        y = ops.linear_act(leaf, w, bias, act, res)
        z = x.double() @ w.double().t() + (0 if bias is None else bias.double())
        want = ACTS[act](z) + (0 if res is None else res.double())
        # as in _check
        zerr = _sum_err(k) * (x.double().abs() @ w.double().abs().t() + (0 if bias is None else bias.double().abs())) + 4 * H
        tol = 1.2 * zerr + 12 * H * (1 + want.abs()) + HALF[dtype] * 1.01 * want.abs() + TINY[dtype]
        assert ((y.detach().double() - want).abs() <= tol).all()
        with torch.no_grad():
            assert torch.equal(ops.linear_act(x, w, bias, act, res), y)
        gy = torch.ones_like(y)                            # what was kept gives the derivative: a bias gradient that is a plain sum of it
        if bias is not None and bias.dtype == torch.float32 and act != "relu":
            lb = bias.clone().requires_grad_(True)
            gb, = torch.autograd.grad(ops.linear_act(x, w, lb, act, res), lb, gy)
            zl = z.clone().requires_grad_(True)
            da, = torch.autograd.grad(ACTS[act](zl).sum(), zl)
            assert ((gb.double() - da.sum(0)).abs() <= (1.2 * zerr + 16 * H).sum(0) + _sum_err(m) * da.abs().sum(0)).all()


@gpu
@pytest.mark.parametrize("act", ["none", "silu", "gelu"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("which,edge,cut,m,k,n", BACK16)
def test_gradients_in_larger_tiles(which, edge, cut, m, k, n, dtype, act):
    got = _plan(dtype, m, k, n, act, which)
    assert got[0] == edge and (got[1] > 1) == cut
    x, w, b, _, gy = _inputs(m, k, n, dtype, torch.float32, 67, residual=False)
    _poison(dtype)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    got = torch.autograd.grad(ops.linear_act(*leaves, activation=act), leaves, gy)
    z = (x.double() @ w.double().t() + b.double()).requires_grad_(True)
    gz = gy.double() * torch.autograd.grad(ACTS[act](z).sum(), z)[0]
    e, tiny = HALF[dtype], TINY[dtype]
    zerr = _sum_err(k) * (x.double().abs() @ w.double().abs().t() + b.double().abs()) + 4 * H
    gzerr = gy.double().abs() * (1.2 * zerr + 16 * H) + e * e * gz.abs() + (2.0 ** -36 if dtype == torch.float16 else 0)
    want, terms = (gz @ w.double(), gz.t() @ x.double()), (_sum_err(2 * n) * (gz.abs() @ w.double().abs()), _sum_err(2 * m) * (gz.abs().t() @ x.double().abs()))
    for a, c, err, t in zip(got, want, (gzerr @ w.double().abs(), gzerr.t() @ x.double().abs()), terms):
        assert ((a.double() - c).abs() <= err + t + e * 1.01 * c.abs() + tiny).all()
        assert (a.double() - c).norm() <= 1.05 * (c.to(dtype).double() - c).norm()
    assert ((got[2].double() - gz.sum(0)).abs() <= (gy.double().abs() * (1.2 * zerr + 16 * H)).sum(0) + _sum_err(m) * gz.abs().sum(0)).all()
    only, = torch.autograd.grad(ops.linear_act(*leaves, activation=act), [leaves[which - 1]], gy)
    assert torch.equal(only, got[which - 1])               # the product by itself


@gpu
@pytest.mark.parametrize("which,m,k,n", WIDE32)
def test_32_bit_products_in_larger_tiles(which, m, k, n):
    act = ("silu", "gelu", "none")[(m + k) % 3]
    assert _plan(torch.float32, m, k, n, act, which)[0] == 128
    _poison(torch.float32)
    _check(*_inputs(m, k, n, torch.float32, torch.float32, 71, residual=m % 2 == 0), act)


def test_plans_cover_every_edge():
    """What the tests above run: every edge whole and cut, but for 256 in the forward product and gx, which the rule does not cut."""
    for dtype in (torch.float16, torch.bfloat16):
        assert {c[:3] for c in WIDE16} == {(0, 128, False), (0, 128, True), (0, 256, False)}
        assert {c[:3] for c in BACK16} == {(w, e, c) for w in (1, 2) for e in (128, 256) for c in (False, True)} - {(1, 256, True)}
        for which, edge, cut, m, k, n in WIDE16 + BACK16:
            assert all(s % 64 for s in (m, k, n))
            for act in ("none", "silu"):
                p = _plan(dtype, m, k, n, act, which)
                assert p[0] == edge and (p[1] > 1) == cut
    for which in range(3):
        assert {(_plan(torch.float32, m, k, n, "none", w)[1] > 1) for w, m, k, n in WIDE32 if w == which} == {False, True}
    assert _plan(torch.float16, 3, 64, 64, "none", 0) == (1, 1) and _plan(torch.float16, 0, 64, 64, "none", 0) == (0, 0)


@gpu
def test_parts_of_more_than_two_to_the_31_elements():
    """gz in two parts of 2.7e9 elements each: rows at both ends of it, all others without a gradient."""
    M, K, N, dtype = 2 ** 26 + 70, 8, 40, torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(3)
    ends = torch.cat([torch.arange(200), torch.arange(M - 200, M)]).cuda()
    x = torch.zeros((M, K), dtype=dtype, device="cuda")
    x[ends] = torch.randn((400, K), generator=g, device="cuda").to(dtype)
    w = torch.randn((N, K), generator=g, device="cuda").to(dtype)
    gy = torch.zeros((M, N), dtype=dtype, device="cuda")
    gy[ends] = torch.randn((400, N), generator=g, device="cuda").to(dtype)
    leaves = [x.requires_grad_(True), w.clone().requires_grad_(True)]
    gx, gw = torch.autograd.grad(ops.linear_act(*leaves, activation="silu"), leaves, gy)
    _, want, _ = _gradients(x.detach()[ends], w, gy[ends], "silu")
    for a, c in ((gx[ends], want[0]), (gw, want[1])):
        assert (a.double() - c).norm() <= 1.05 * (c.to(dtype).double() - c).norm()
    assert not gx[200:100000].any() and not gx[-100000:-200].any()


def test_c_entry_refuses_a_kept_z_that_is_not_aligned():
    """It is written 16 bytes at a time."""
    from sound_event_detection_dcase2017_task4_amd import _lib
    for z in (2, 4, 24):
        assert _lib.lib().sed_linear_fwd(16, 16, None, None, 1, 1, 100, 8, 8, 2, 16, z, None, 0, None) == -22
