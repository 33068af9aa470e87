"""optim.FusedAdamW (sed_adamw): against the definition in 64 bits, the 8-bit codes bit for bit against the same 32-bit operations in
numpy, and its refusals.  Tolerances count roundings: an operation in 32 bits is off by at most H = 2^-24 relative to its result."""
import numpy as np
import pytest
import torch

from sound_event_detection_dcase2017_task4_amd import ops, optim

H = 2.0 ** -24
SIZES = [1, 3, 255, 256, 257, 1023, 4095, 4096, 4097, 20001]
gpu = pytest.mark.gpu


def _tensors(sizes, dtypes, seed, shift=0):
    """Parameters (shift > 0: that many elements into a buffer, so that they are not aligned) with gradients over many decades."""
    g = torch.Generator().manual_seed(seed)
    ps = []
    for k, n in enumerate(sizes):
        t = dtypes[k % len(dtypes)]
        data, grad = torch.randn(n + shift, generator=g) * 0.05, torch.randn(n + shift, generator=g)
        grad *= torch.exp(2.0 * torch.randn(n + shift, generator=g)) * 0.01
        p = torch.nn.Parameter(data.to(t).cuda()[shift:])
        p.grad = grad.to(t).cuda()[shift:]
        ps.append(p)
    return ps


def _flat(opt, values):
    out = torch.zeros(opt.exp_avg.numel(), dtype=torch.float64)
    for at, v in zip(opt.offsets, values):
        out[at:at + v.numel()] = v.detach().double().cpu().reshape(-1)
    return out


def _reference(p, g, m, v, t, lr, b1, b2, eps, wd):
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    p = p * (1 - lr * wd) - lr / (1 - b1 ** t) * m / (torch.sqrt(v / (1 - b2 ** t)) + eps)
    return p, m, v


@gpu
@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("dtypes", [(torch.float32,), (torch.bfloat16,), (torch.float16, torch.float32, torch.bfloat16)])
def test_32_bit_moments_against_64_bits(dtypes, shift):
    ps = _tensors(SIZES, dtypes, 3, shift)
    lr, betas, eps, wd, T = 3e-3, (0.9, 0.99), 1e-7, 0.1, 4
    opt = optim.FusedAdamW([{"params": ps[:4]}, {"params": ps[4:], "weight_decay": 0.0, "lr": 1e-2}], lr=lr, betas=betas, eps=eps, weight_decay=wd)
    want = [(p.detach().double(), torch.zeros(p.shape, dtype=torch.float64, device="cuda"), torch.zeros(p.shape, dtype=torch.float64, device="cuda"))
            for p in ps]
    for t in range(1, T + 1):
        for k, p in enumerate(ps):
            p.grad.mul_(-0.7)
            a = (lr, *betas, eps, wd) if k < 4 else (1e-2, *betas, eps, 0.0)
            want[k] = _reference(want[k][0], 0.5 * p.grad.double(), want[k][1], want[k][2], t, *a)
        opt.step(grad_scale=0.5)
    m, v = opt.moments()
    for k, p in enumerate(ps):
        at, n = opt.offsets[k], p.numel()
        wp, wm, wv = want[k]
        # a moment: two constants and three operations a step, over T steps.  The terms of m may cancel: relative to the largest |g| so far
        assert (m[at:at + n].double() - wm).abs().le(T * 5 * H * (p.grad.double().abs() * 0.5 / 0.7 ** T)).all()
        assert (v[at:at + n].double() - wv).abs().le(T * 6 * H * wv).all()
        # the parameter: T roundings of itself and of the decay, and an update of at most lr / c1 * |m| / sqrt(v / c2) <= 8 lr here
        # with the errors of m (relative to the largest term: 4), v, the division, the root and the constants (12)
        got = p.detach().double() if p.dtype == torch.float32 else opt.master[opt._copy_at[k]:opt._copy_at[k] + n].double()
        a = (lr, wd) if k < 4 else (1e-2, 0.0)
        assert (got - wp).abs().le(T * (4 * H * (wp.abs() + 8 * a[0]) + 40 * H * 8 * a[0])).all()
        if p.dtype != torch.float32:
            assert torch.equal(p.detach(), got.float().to(p.dtype))       # the copy, rounded once


def _np_decode(opt):
    f = np.float32
    q, s = opt.exp_avg.cpu().numpy().astype(f), np.repeat(opt.exp_avg_scale.cpu().numpy(), 256)
    u = q * f(1.0 / 127.0)
    m = u * np.abs(u) * s
    q, s = opt.exp_avg_sq.cpu().numpy().astype(f), np.repeat(opt.exp_avg_sq_scale.cpu().numpy(), 256)
    u = q * f(1.0 / 255.0)
    u = u * u
    return m, u * u * s


@gpu
@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("dtypes", [(torch.float32,), (torch.float16, torch.float32, torch.bfloat16)])
def test_8_bit_moments_bit_for_bit(dtypes, shift):
    ps = _tensors(SIZES, dtypes, 7, shift)
    lr, (b1, b2), eps, wd = 3e-3, (0.9, 0.99), 1e-7, 0.1
    opt = optim.FusedAdamW(ps, lr=lr, betas=(b1, b2), eps=eps, weight_decay=wd, state_bits=8)
    f = np.float32
    for t in range(1, 5):
        for p in ps:
            p.grad.mul_(-0.7)
        m, v = _np_decode(opt)
        got = opt.moments()
        assert np.array_equal(got[0].cpu().numpy(), m) and np.array_equal(got[1].cpu().numpy(), v)
        p0 = _flat(opt, [p if p.dtype == torch.float32 or t == 1 else opt.master[c:c + p.numel()] for p, c in zip(ps, opt._copy_at)])
        g = _flat(opt, [p.grad for p in ps]).numpy().astype(f)
        opt.step()
        m = m * f(b1) + g * f(1.0 - b1)
        v = v * f(b2) + g * g * f(1.0 - b2)
        sm, sv = np.abs(m).reshape(-1, 256).max(1), v.reshape(-1, 256).max(1)
        assert np.array_equal(opt.exp_avg_scale.cpu().numpy(), sm) and np.array_equal(opt.exp_avg_sq_scale.cpu().numpy(), sv)
        dm, dv = np.repeat(np.where(sm > 0, sm, 1), 256).astype(f), np.repeat(np.where(sv > 0, sv, 1), 256).astype(f)
        qm = np.rint(np.sqrt(np.abs(m) / dm) * f(127))
        qv = np.rint(np.sqrt(np.sqrt(v / dv)) * f(255))
        qv = np.where(v > 0, np.maximum(qv, 1), qv)
        assert np.array_equal(opt.exp_avg.cpu().numpy(), np.where(m < 0, -qm, qm).astype(np.int8))
        assert np.array_equal(opt.exp_avg_sq.cpu().numpy(), qv.astype(np.uint8))
        # the parameter takes the moments before they are rounded to 8 bits: one step of 64-bit arithmetic on them
        w = p0 * (1 - lr * wd) - lr / (1 - b1 ** t) * torch.from_numpy(m).double() / (torch.sqrt(torch.from_numpy(v).double() / (1 - b2 ** t)) + eps)
        after = _flat(opt, [p if p.dtype == torch.float32 else opt.master[c:c + p.numel()] for p, c in zip(ps, opt._copy_at)])
        assert (after - w).abs().le(4 * H * w.abs() + 20 * H * (w - p0).abs()).all()


@gpu
def test_8_bit_codes_are_near_what_they_stand_for():
    """Half a step of the root's grid on either side: |m - decoded| <= scale (|q| + 1/4) / 127^2, and sqrt(v) likewise on 255; a positive
    second moment never reads back as zero.  A few roundings of 32 bits come on top."""
    n = 256 * 64
    p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
    g = torch.Generator().manual_seed(1)
    p.grad = (torch.randn(n, generator=g) * torch.exp(3 * torch.randn(n, generator=g))).cuda()
    p.grad[5], p.grad[300:512] = 0.0, 0.0
    opt = optim.FusedAdamW([p], betas=(0.0, 0.0), state_bits=8)         # the moments are g and g^2 themselves
    opt.step()
    m, v = (x.double() for x in opt.moments())
    gd, s = p.grad.double(), opt.exp_avg_scale.double().repeat_interleave(256)
    q = opt.exp_avg.double().abs()
    assert (m - gd).abs().le(s * ((q + 0.25) / 127 ** 2) + 16 * H * s).all()
    r, root, sv = v.sqrt(), gd.abs(), opt.exp_avg_sq_scale.double().repeat_interleave(256).sqrt()
    q = opt.exp_avg_sq.double()
    assert (r - root).abs().le(sv * ((q + 0.25) / 255 ** 2) + 16 * H * sv)[q > 1].all()
    assert ((v > 0) == (p.grad * p.grad > 0)).all() and v[5] == 0 and m[5] == 0


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_tensors_without_gradient_and_padding_stay(bits):
    ps = _tensors([300, 70, 5000], (torch.float32, torch.bfloat16), 11)
    opt = optim.FusedAdamW(ps, state_bits=bits)
    opt.step()
    ps[1].grad = None
    before = [p.detach().clone() for p in ps]
    m0, v0 = (x.clone() for x in opt.moments())
    opt.step()
    m1, v1 = opt.moments()
    lo, hi = opt.offsets[1], opt.offsets[2]
    assert torch.equal(before[1], ps[1].detach()) and torch.equal(m0[lo:hi], m1[lo:hi]) and torch.equal(v0[lo:hi], v1[lo:hi])
    assert not torch.equal(before[0], ps[0].detach()) and not torch.equal(before[2], ps[2].detach())
    used = torch.zeros(m1.numel(), dtype=torch.bool, device="cuda")
    for at, p in zip(opt.offsets, ps):
        used[at:at + p.numel()] = True
    assert not m1[~used].any() and not v1[~used].any()
    for p in ps:
        p.grad = None
    opt.step()                                                    # nothing to do at all
    assert torch.equal(m1, opt.moments()[0])


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_nan_and_infinity_stay_where_they_are(bits):
    p = torch.nn.Parameter(torch.ones(1024, device="cuda"))
    p.grad = torch.full((1024,), 0.1, device="cuda")
    p.grad[300], p.grad[700] = float("nan"), float("inf")
    opt = optim.FusedAdamW([p], state_bits=bits)
    opt.step()
    bad = torch.zeros(1024, dtype=torch.bool, device="cuda")
    bad[300] = bad[700] = True                                    # inf / inf is NaN as well
    assert torch.equal(torch.isnan(p.detach()), bad)
    m, v = opt.moments()
    if bits == 8:                                                 # the scale is the block's: the block reads back as NaN, its neighbours do not
        bad[256:512] = bad[512:768] = True
    assert torch.equal(~torch.isfinite(m), bad) and torch.equal(~torch.isfinite(v), bad)


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict_continues_bit_for_bit(bits):
    make = lambda: _tensors([1000, 257, 64], (torch.float32, torch.float16), 5)  # noqa: E731
    a, b = make(), make()
    oa, ob = optim.FusedAdamW(a, state_bits=bits), optim.FusedAdamW(b, state_bits=bits)
    for _ in range(3):
        oa.step()
    for x, y in zip(a, b):
        y.data.copy_(x.data)
    sd = {k: (v.cpu() if torch.is_tensor(v) else v) for k, v in oa.state_dict().items()}
    ob.load_state_dict(sd)
    for _ in range(2):
        oa.step()
        ob.step()
    for x, y in zip(a, b):
        assert torch.equal(x.detach(), y.detach())
    assert ob.step_count == 5 and torch.equal(oa.exp_avg, ob.exp_avg) and torch.equal(oa.exp_avg_sq, ob.exp_avg_sq)
    for change in ({"state_bits": 40 - bits}, {"exp_avg": sd["exp_avg"][:-256]}, {"numels": [1, 2, 3]}, {"exp_avg_sq": None},
                   {"exp_avg": sd["exp_avg"].double()}, {"step": -1}):
        with pytest.raises(ValueError):
            ob.load_state_dict(dict(sd, **change))
    with pytest.raises(ValueError):
        ob.load_state_dict({"state": {}, "param_groups": []})
    assert ob.step_count == 5 and torch.equal(oa.exp_avg, ob.exp_avg)


@gpu
def test_copy_follows_a_parameter_that_torch_changed():
    p = torch.nn.Parameter(torch.ones(300, device="cuda", dtype=torch.bfloat16))
    p.grad = torch.zeros_like(p)
    opt = optim.FusedAdamW([p], weight_decay=0.0)
    opt.step()
    with torch.no_grad():
        p.mul_(3.0)
    opt.step()
    assert torch.equal(p.detach(), torch.full_like(p, 3.0)) and float(opt.master[0]) == 3.0
    p.data = torch.full((300,), 7.0, device="cuda", dtype=torch.bfloat16)          # moved as well
    p.grad = torch.zeros_like(p)
    opt.step()
    assert float(opt.master[0]) == 7.0 and torch.equal(p.detach(), torch.full_like(p, 7.0))


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bits", [32, 8])
def test_copy_follows_a_parameter_that_was_written_through_data(dtype, bits):
    """A write that no version counter records: elements that are not the rounding of their copy are taken, the others keep their bits."""
    p = torch.nn.Parameter(torch.linspace(-2.0, 2.0, 1001, device="cuda").to(dtype)[1:])          # 16-bit vectors begin beside 8 bytes
    p.grad = torch.full_like(p, 0.3)
    opt = optim.FusedAdamW([p], lr=1e-3, weight_decay=0.0, state_bits=bits)
    for _ in range(3):
        opt.step()
    kept = opt.master[:1000].clone()
    assert torch.equal(kept.to(dtype), p.detach()) and not torch.equal(kept.to(dtype).float(), kept)
    p.data[100:200] = 5.0
    p.data[300] = float("nan")
    p.grad.zero_()
    opt.param_groups[0]["lr"] = 0.0
    assert float(opt.state_dict()["master"][150]) == 5.0
    opt.master[:1000] = kept                               # the step does the same by itself
    opt.step()
    want = kept.clone()
    want[100:200] = 5.0
    want[300] = float("nan")
    assert torch.equal(opt.master[:1000].nan_to_num(99.0), want.nan_to_num(99.0))
    assert torch.equal(p.detach().nan_to_num(99.0), want.to(dtype).nan_to_num(99.0))


@gpu
def test_gradients_of_any_layout_moved_between_steps_and_other_streams():
    p, q = (torch.nn.Parameter(torch.ones(33, 40, device="cuda")) for _ in range(2))
    grads = [torch.randn(40, 33, device="cuda").t() for _ in range(4)]
    a, b = optim.FusedAdamW([p]), optim.FusedAdamW([q])
    side = torch.cuda.Stream()
    for k, g in enumerate(grads):
        p.grad, q.grad = g, g.contiguous()
        a.step()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side if k % 2 else torch.cuda.current_stream()):
            b.step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
    assert torch.equal(p.detach(), q.detach())


@gpu
def test_refused_step_is_taken_back():
    p = torch.nn.Parameter(torch.ones(300, device="cuda"))
    p.grad = torch.ones_like(p)
    opt = optim.FusedAdamW([p])
    opt.step()
    before, m = p.detach().clone(), opt.exp_avg.clone()
    ops._err_dev(p.device)[0] = 1                                  # as a split-f16 kernel leaves it behind a NaN operand
    torch.cuda.synchronize()
    ops._err_flag()[1] = 1
    with pytest.raises(ops.NonFiniteOperand) as e:
        opt.step()
    assert e.value.skipped_steps == 1 and opt.step_count == 1 and opt.skipped_steps == 1
    assert torch.equal(before, p.detach()) and torch.equal(m, opt.exp_avg)
    opt.step()
    assert opt.step_count == 2 and not torch.equal(before, p.detach())


@gpu
def test_step_refuses_capture_and_follows_a_replay():
    w = torch.nn.Parameter(torch.ones(300, device="cuda"))
    x = torch.randn(300, device="cuda")
    opt = optim.FusedAdamW([w])
    w.grad = torch.zeros_like(w)
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    refused = []
    with torch.cuda.stream(side):
        graph.capture_begin()
        try:
            w.grad.copy_(x)
            try:
                opt.step()
            except RuntimeError as e:
                refused.append(str(e))
        finally:
            graph.capture_end()
    torch.cuda.current_stream().wait_stream(side)
    assert len(refused) == 1 and "captured" in refused[0] and opt.step_count == 0
    v = torch.nn.Parameter(torch.ones(300, device="cuda"))
    other = optim.FusedAdamW([v])
    for k in range(3):
        x.normal_()
        graph.replay()
        opt.step()
        v.grad = x.clone()
        other.step()
        torch.cuda.synchronize()
        assert torch.equal(w.detach(), v.detach()), k


@gpu
def test_more_than_two_to_the_31_elements():
    n = 2 ** 31 + 300
    p = torch.nn.Parameter(torch.zeros(n, dtype=torch.float16, device="cuda"))
    p.grad = torch.zeros(n, dtype=torch.float16, device="cuda")
    p.grad[-300:] = 1.0
    p.grad[5] = 1.0
    opt = optim.FusedAdamW([p], lr=0.5, weight_decay=0.0, state_bits=8)
    opt.step()
    assert torch.equal(p.detach()[-300:], torch.full((300,), -0.5, dtype=torch.float16, device="cuda")) and float(p.detach()[5]) == -0.5
    assert not p.detach()[6:100000].any() and not p.detach()[-100000:-300].any()
    assert int((opt.exp_avg[:n] != 0).sum()) == 301


@gpu
def test_refusals_on_the_gpu():
    p = torch.nn.Parameter(torch.ones(4, 6, device="cuda"))
    for bad in ([p, p], [torch.nn.Parameter(p.data[:2]), torch.nn.Parameter(p.data[1:])], [torch.nn.Parameter(p.data.t())],
                [torch.nn.Parameter(p.data.double())]):
        with pytest.raises(ValueError):
            optim.FusedAdamW(bad)
    with pytest.raises(RuntimeError):
        optim.FusedAdamW([p, torch.nn.Parameter(torch.ones(3))])
    flat = optim.FusedAdamAmsgrad([torch.nn.Parameter(torch.ones(8, device="cuda"))], lr=1e-3)
    with pytest.raises(ValueError):
        optim.FusedAdamW(flat.params)
    opt = optim.FusedAdamW([p])
    p.grad = torch.ones_like(p)
    opt.step()
    for smaller in (torch.ones(5, 6, device="cuda"), p.data[:2]):      # the second one at the same address
        p.data = smaller
        p.grad = None
        p.grad = torch.ones_like(p)
        with pytest.raises(ValueError):
            opt.step()
    assert opt.step_count == 1


def test_refusals_on_the_cpu():
    p = torch.nn.Parameter(torch.ones(4))
    for kw in ({"state_bits": 16}, {"betas": (1.0, 0.9)}, {"betas": (0.9, -0.1)}, {"lr": -1.0}, {"eps": -1e-8}, {"weight_decay": -0.1}):
        with pytest.raises(ValueError):
            optim.FusedAdamW([p], **kw)
    for bad in ([], [{"params": [p], "momentum": 0.9}], [{"params": [torch.nn.Parameter(torch.ones(1))]} for _ in range(17)]):
        with pytest.raises(ValueError):
            optim.FusedAdamW(bad)
    with pytest.raises(RuntimeError):
        optim.FusedAdamW([p])


def test_c_entries_refuse_bad_arguments():
    from sound_event_detection_dcase2017_task4_amd import _lib
    h = _lib.lib()
    ok = (1e-3, 0.9, 0.999, 1e-8, 0.01)

    def call(rows=1, chunks=1, n=1, m=1, ms=1, bits=32, hyper=ok, groups=1, step=1, flag=None, skipped=None):
        hy = np.array(hyper, dtype=np.float64)
        return h.sed_adamw(rows, chunks, n, m, 1, ms, ms, None, bits, hy.ctypes.data, groups, step, 1.0, flag, skipped, None)
    for bad in ({"rows": None}, {"chunks": None}, {"n": 0}, {"n": 1 << 31}, {"m": None}, {"bits": 16}, {"bits": 8, "ms": None}, {"groups": 0},
                {"groups": 17}, {"step": 0}, {"hyper": (1e-3, 1.0, 0.9, 0.0, 0.0)}, {"hyper": (1e-3, 0.9, 0.9, -1.0, 0.0)}, {"flag": 1}):
        assert call(**bad) == -22, bad
    assert h.sed_adamw_moments(1, 1, 1, 1, 255, 1, 1, None) == -22 and h.sed_adamw_moments(1, 1, 1, 1, 0, 1, 1, None) == -22
    assert h.sed_adamw_moments(1, None, 1, 1, 256, 1, 1, None) == -22 and h.sed_adamw_chunk() % 256 == 0


def _model(seed=5):
    from oracle import model as om
    from sound_event_detection_dcase2017_task4_amd.pytorch import models
    m = models.Cnn_9layers_FrameAvg(32000, 1024, 320, 64, 50, 14000, 17)
    m.load_state_dict(om.recipe_state("Cnn_9layers_FrameAvg", seed))
    rs = np.random.RandomState(seed)
    x, y = torch.from_numpy((rs.randn(4, 32000) * 0.1).astype(np.float32)).cuda(), torch.from_numpy((rs.rand(4, 17) < 0.2).astype(np.float32)).cuda()
    return m.cuda().train(), x, y


def _report():
    """As a split-f16 kernel that met a NaN operand leaves the two words."""
    ops._err_dev()[0] = 1
    torch.cuda.synchronize()
    ops._err_flag()[1] = 1


def _statistics(m):
    return {k: v.clone() for k, v in m.named_buffers() if "running" in k}


@gpu
@pytest.mark.parametrize("passes", [1, 2])
def test_refused_step_takes_the_batchnorm_statistics_back(passes):
    """Clean forward passes install their statistics; behind them a kernel reports an operand that is not finite, and the step is refused."""
    from sound_event_detection_dcase2017_task4_amd.pytorch.losses import clip_bce
    m, x, y = _model()
    opt = optim.FusedAdamW(m, lr=1e-3)
    ops.check_device_errors(synchronize=True)

    def step(reported=False):
        opt.zero_grad()
        for k in range(passes):
            clip_bce(m(x * (1 + k)), {"target": y}).backward()
        if reported:
            _report()
        opt.step()
        ops.check_device_errors(synchronize=True)
    for _ in range(2):
        step()
        assert ops._BN_LAST is None                               # nothing of a settled step is kept
    before, stats = [p.detach().clone() for p in opt.params], _statistics(m)
    with pytest.raises(ops.NonFiniteOperand):
        step(reported=True)
    assert opt.step_count == 2 and opt.skipped_steps == 1
    assert all(torch.equal(p.detach(), b) for p, b in zip(opt.params, before))
    assert all(torch.equal(v, stats[k]) for k, v in _statistics(m).items())
    ops.rollback_bn_counters(m, passes)
    step()
    assert opt.step_count == 3 and not torch.equal(m.bn0.running_mean, stats["bn0.running_mean"])


@gpu
def test_a_refused_step_of_the_other_optimiser_leaves_the_statistics_of_settled_steps():
    from sound_event_detection_dcase2017_task4_amd.pytorch.losses import clip_bce
    m, x, y = _model()
    opt = optim.FusedAdamW(m, lr=1e-3)
    ops.check_device_errors(synchronize=True)
    for _ in range(2):
        opt.zero_grad()
        clip_bce(m(x), {"target": y}).backward()
        opt.step()
    stats = _statistics(m)
    other, x2, y2 = _model(6)
    flat = optim.FusedAdamAmsgrad(other, lr=1e-3)
    flat.zero_grad()
    clip_bce(other(x2), {"target": y2}).backward()
    _report()
    with pytest.raises(ops.NonFiniteOperand):
        flat.step()
        ops.check_device_errors(synchronize=True)
    assert all(torch.equal(v, stats[k]) for k, v in _statistics(m).items())


@gpu
def test_lagged_poll_reports_a_refused_step_two_steps_later():
    p = torch.nn.Parameter(torch.ones(300, device="cuda"))
    p.grad = torch.ones_like(p)
    opt = optim.FusedAdamW([p], poll_lag=2)
    ops.check_device_errors(synchronize=True)
    opt.step()
    before = p.detach().clone()
    _report()
    opt.step()
    opt.step()
    with pytest.raises(ops.NonFiniteOperand) as e:
        opt.step()
    assert e.value.skipped_steps == 3 and opt.step_count == 1 and opt.skipped_steps == 3 and torch.equal(before, p.detach())
    opt.step()
    opt.poll(0)
    assert opt.step_count == 2 and not torch.equal(before, p.detach())


def test_guard_collect_refuses_bad_arguments():
    from sound_event_detection_dcase2017_task4_amd import _lib
    h = _lib.lib()
    assert h.sed_guard_collect(16, None, 16, None, None, None) == -22 and h.sed_guard_collect(16, 16, None, None, 16, None) == -22


@gpu
def test_changed_groups_are_refused():
    ps = [torch.nn.Parameter(torch.ones(300, device="cuda")) for _ in range(4)]
    for p in ps:
        p.grad = torch.ones_like(p)
    opt = optim.FusedAdamW([{"params": ps[:1]}, {"params": ps[1:3], "lr": 1e-2}])
    opt.step()
    before = [p.detach().clone() for p in ps]
    groups = [dict(g, params=list(g["params"])) for g in opt.param_groups]
    for changed in (groups[:1], groups + [{**groups[0], "params": ps[3:]}], [groups[0], {**groups[1], "params": ps[1:]}], groups[::-1],
                    [{**groups[0], "params": ps[3:]}, groups[1]], [{**groups[0], "params": ps[:2]}, {**groups[1], "params": ps[2:3]}], []):
        opt.param_groups = changed
        with pytest.raises(ValueError, match="groups"):
            opt.step()
    assert opt.step_count == 1 and all(torch.equal(p.detach(), b) for p, b in zip(ps, before))
    groups[1]["lr"] = 0.5                                         # an option may change
    opt.param_groups = groups
    opt.step()
    assert opt.step_count == 2 and float((ps[1].detach() - before[1]).abs().min()) > 0.1


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_state_without_copies_takes_them_from_the_parameters(bits):
    ps = _tensors([1000, 257], (torch.bfloat16, torch.float32, torch.float16), 5)
    opt = optim.FusedAdamW(ps, state_bits=bits)
    for _ in range(3):
        opt.step()
    p = ps[0].detach().float().reshape(-1)
    assert not torch.equal(opt.master[:1000], p)                  # the copy has bits that its rounding has not
    sd = opt.state_dict()
    for state in (dict(sd, master=None), {k: v for k, v in sd.items() if k != "master"}):
        kept = opt.master.clone()
        opt.load_state_dict(state)
        assert torch.equal(opt.master[:1000], p)
        opt.load_state_dict(dict(sd, master=kept))
        assert torch.equal(opt.master, kept)
