"""Operators of a residual block on channels-last activations, and of the optimiser that trains it: group normalisation with an
activation, the matrix product with bias, activation and residual in its epilogue, and the AdamW step over many tensors.

A case is a dict of plain values.  `prepare` makes what a program has in hand, `run` is one pass through the operator: its plain
form in elementary torch operations (own = False), or the calls of this package (own = True).  `exact` is the definition in 64 bits.
"""
import itertools
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}
BLOCK = 256                     # elements that share one scale of an 8-bit optimiser state; every tensor's state starts a block
EPS = 1e-5                      # of the normalisation


# ---------------------------------------------------------------------------------------------------------------- the cases

def _norm(name, dtype, batch, rows, channels, groups, act, train):
    return {"name": name, "op": "norm", "dtype": dtype, "batch": batch, "rows": rows, "channels": channels, "groups": groups,
            "act": act, "train": train}


def _linear(name, dtype, m, k, n, act, residual, train):
    return {"name": name, "op": "linear", "dtype": dtype, "m": m, "k": k, "n": n, "act": act, "residual": residual, "train": train}


def _adamw(name, dtype, bits, tensors, total, seed):
    return {"name": name, "op": "adamw", "dtype": dtype, "bits": bits, "tensors": tensors, "total": total, "shapes": seed}


def listed():
    return [
        # the frame features behind the trunk (125 frames x 512 channels) of four clips: a launch-bound inference call
        _norm("norm_frames_fp32", "fp32", 4, 125, 512, 32, "none", False),
        # the second ConvBlock at the batch of the headline run, 500 x 32 positions x 128 channels, forward and backward
        _norm("norm_block2_train_bf16", "bf16", 32, 16000, 128, 32, "silu", True),
        # an odd number of channels and rows: three channels a group, no 16-byte alignment of a row
        _norm("norm_odd_train_fp32", "fp32", 3, 5661, 51, 17, "gelu", True),
        # the first ConvBlock over a whole batch of 256 clips: the largest activation of the models, inference
        _norm("norm_block1_fp16", "fp16", 256, 64064, 64, 8, "silu", False),
        # one frame through the first product of a feed-forward pair, as a streaming detector asks for it
        _linear("linear_frame_bf16", "bf16", 1, 512, 2048, "gelu", False, False),
        # sixteen streams at once through the second product, with the residual
        _linear("linear_streams_fp16", "fp16", 16, 2048, 512, "none", True, False),
        # the headline batch (32 clips x 125 frames) through the first product, forward and backward
        _linear("linear_frames_train_bf16", "bf16", 4000, 512, 2048, "gelu", False, True),
        # odd sizes in 32 bits: rows that are not 16-byte aligned, tiles that end inside the matrix
        _linear("linear_odd_train_fp32", "fp32", 1001, 513, 127, "silu", True, True),
        # 256 clips x 125 frames through a wide product with everything in the epilogue, forward and backward
        _linear("linear_wide_train_bf16", "bf16", 32000, 2048, 2048, "silu", True, True),
        # the parameters of the nine-layer models: 28 tensors from 17 elements to 2.4 million
        _adamw("adamw_model_fp32", "fp32", 32, 28, 4700000, 1),
        # a 16-bit model with a 32-bit copy of its weights, tensors of odd sizes
        _adamw("adamw_copy_bf16", "bf16", 32, 37, 30000001, 2),
        # a large model with its two states in 8 bits
        _adamw("adamw_large_8bit", "fp32", 8, 60, 240000000, 3),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("norm", "norm", "linear", "linear", "linear", "adamw", "adamw"))
    if op == "norm":
        groups = _log(rng, 1, 64)
        channels = groups * _log(rng, 1, 1024 // groups)
        batch = _log(rng, 1, 256)
        rows = _log(rng, max(1, -(-16 * groups // channels)), max(32, min(64064, 200000000 // (batch * channels))))
        train = rng.random() < 0.6
        # the gradient of ReLU jumps at zero, where the last bit of a sum decides: ReLU is drawn for forward passes
        c = _norm("", rng.choice(list(DTYPES)), batch, rows, channels, groups,
                  rng.choice(("none", "silu", "gelu") if train else ("none", "relu", "silu", "gelu")), train)
    elif op == "linear":
        k, n = _log(rng, 16, 4096), _log(rng, 16, 4096)
        m = _log(rng, 1, 32000)
        if rng.random() < 0.6:                       # most widths of real layers are multiples of 8, not all are
            k, n = -(-k // 8) * 8, -(-n // 8) * 8
        m = max(1, min(m, int(1.3e11 / (k * n))))
        train = rng.random() < 0.5
        c = _linear("", rng.choice(list(DTYPES)), m, k, n, rng.choice(("none", "silu", "gelu") if train else ("none", "relu", "silu", "gelu")),
                    rng.random() < 0.5, train)
    else:
        dtype = rng.choice(list(DTYPES))
        c = _adamw("", dtype, rng.choice((8, 32)), rng.randint(1, 60), _log(rng, 20000, 200000000), rng.randint(10, 99999))
    del c["name"]
    return c


def _sizes(case):
    """Element counts of the tensors of an AdamW case: a few large, many small, with odd ones among them."""
    g = torch.Generator().manual_seed(case["shapes"])
    share = torch.exp(2.0 * torch.randn((case["tensors"],), generator=g, dtype=torch.float64))
    n = (share / share.sum() * case["total"]).long().clamp_min(1)
    n[n > 4096] -= n[n > 4096] % 8                    # matrices; the small ones (vectors) keep their odd sizes
    return [int(v) for v in n]


def _decayed(case):
    """How many of the tensors, the first ones, take weight decay."""
    return (case["tensors"] + 1) // 2


# ---------------------------------------------------------------------------------------------------------------- inputs

def _hyper():
    return {"lr": 1e-3, "betas": (0.9, 0.999), "eps": 1e-8, "weight_decay": 0.01}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype)


def _prepare_norm(case, g):
    t = DTYPES[case["dtype"]]
    B, S, C = case["batch"], case["rows"], case["channels"]
    x = _randn(g, B, S, C, dtype=t)
    x.mul_((0.5 + torch.rand((C,), generator=g, device="cuda")).to(t)).add_((0.5 * _randn(g, C)).to(t))
    s = {"x": x, "weight": 1.0 + 0.2 * _randn(g, C), "bias": 0.2 * _randn(g, C)}
    if case["train"]:
        s["gy"] = _randn(g, B, S, C, dtype=t)
    return s


def _prepare_linear(case, g):
    t = DTYPES[case["dtype"]]
    M, K, N = case["m"], case["k"], case["n"]
    s = {"x": _randn(g, M, K, dtype=t), "weight": (_randn(g, N, K) / math.sqrt(K)).to(t), "bias": (0.1 * _randn(g, N)).to(t),
         "residual": _randn(g, M, N, dtype=t) if case["residual"] else None}
    if case["train"]:
        s["gy"] = _randn(g, M, N, dtype=t)
    return s


def _prepare_adamw(case, g):
    """Parameters and gradients, each as one buffer in which every tensor begins at a multiple of BLOCK elements, and the two
    moments behind a hundred steps: 32-bit values, or their 8-bit codes and scales."""
    t = DTYPES[case["dtype"]]
    sizes = _sizes(case)
    blocks = [-(-n // BLOCK) for n in sizes]
    first = [BLOCK * k for k in itertools.accumulate([0] + blocks)]
    total = first.pop()
    per_block = torch.tensor([n - BLOCK * k for n, b in zip(sizes, blocks) for k in range(b)], device="cuda")
    inside = (torch.arange(BLOCK, device="cuda") < per_block.view(-1, 1)).view(-1)
    master = (0.05 * _randn(g, total)).mul_(inside)
    grad = _randn(g, total).mul_(0.01).mul_(torch.exp(_randn(g, total // BLOCK, 1)).expand(-1, BLOCK).reshape(-1)).mul_(inside)
    m = (0.3 * grad + 0.003 * _randn(g, total)).mul_(inside)
    v = (grad * grad * 0.5 + 1e-5 * torch.rand((total,), generator=g, device="cuda")).mul_(inside)
    decayed = sum(blocks[:_decayed(case)])
    s = {"sizes": sizes, "first": first, "steps": 100, "param": master.to(t), "grad": grad.to(t),
         "master": master if t != torch.float32 else None, "decayed": decayed * BLOCK}
    if case["bits"] == 8:
        s["m"], s["m_scale"] = _encode_m(m)
        s["v"], s["v_scale"] = _encode_v(v)
    else:
        s["m"], s["v"] = m, v
    return s


def prepare(case, seed):
    g = _gen(seed)
    if case["op"] == "norm":
        s = _prepare_norm(case, g)
    elif case["op"] == "linear":
        s = _prepare_linear(case, g)
    else:
        s = _prepare_adamw(case, g)
    s["case"] = case
    if case.get("train"):
        for name in ("x", "weight", "bias", "residual"):
            if s.get(name) is not None:
                s[name].requires_grad_(True)
    if own and case["op"] == "adamw":
        s["optimizer"] = _own_optimizer(s, case)      # the handle that a training program keeps from step to step
    return s


# ---------------------------------------------------------------------------------------------------------------- plain forms

def _act(z, act):
    if act == "relu":
        return z.clamp_min(0.0)
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    return z


def _act_grad(z, act):
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return s * (1.0 + z * (1.0 - s))
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    return torch.ones_like(z)


def _plain_norm(s, case):
    x = s["x"].detach()
    B, S, C = x.shape
    G = case["groups"]
    w, b = s["weight"].detach(), s["bias"].detach()
    xg = x.float().view(B, S, G, C // G)
    d = xg - xg.mean(dim=(1, 3), keepdim=True)
    rstd = 1.0 / torch.sqrt((d * d).mean(dim=(1, 3), keepdim=True) + EPS)
    xhat = (d * rstd).view(B, S, C)
    z = xhat * w + b
    y = _act(z, case["act"]).to(x.dtype)
    if not case["train"]:
        return {"y": y}
    gz = s["gy"].float() * _act_grad(z, case["act"])
    gw, gb = (gz * xhat).sum(dim=(0, 1)), gz.sum(dim=(0, 1))
    gh = (gz * w).view(B, S, G, C // G)
    hg = xhat.view(B, S, G, C // G)
    gx = (gh - gh.mean(dim=(1, 3), keepdim=True) - hg * (gh * hg).mean(dim=(1, 3), keepdim=True)) * rstd
    return {"y": y, "gx": gx.view(B, S, C).to(x.dtype), "gweight": gw, "gbias": gb}


def _plain_linear(s, case):
    t = s["x"].dtype
    x, w, b = s["x"].detach().float(), s["weight"].detach().float(), s["bias"].detach().float()
    z = x @ w.t() + b
    y = _act(z, case["act"])
    if s["residual"] is not None:
        y = y + s["residual"].detach().float()
    y = y.to(t)
    if not case["train"]:
        return {"y": y}
    gz = s["gy"].float() * _act_grad(z, case["act"])
    r = {"y": y, "gx": (gz @ w).to(t), "gweight": (gz.t() @ x).to(t), "gbias": gz.sum(dim=0).to(t)}
    if s["residual"] is not None:
        r["gresidual"] = s["gy"]
    return r


# An 8-bit moment holds, per block of 256 elements, the largest magnitude as a float and per element the code
#   first moment   q = round(127 sqrt(|m| / scale)) with m's sign,   m = sign(q) (|q| / 127)^2 scale
#   second moment  q = round(255 (v / scale)^(1/4)), at least 1 where v > 0,   v = (q / 255)^4 scale
def _encode_m(m):
    m = m.view(-1, BLOCK)
    scale = m.abs().amax(dim=1, keepdim=True)
    q = torch.round(torch.sqrt(m.abs() / torch.where(scale > 0, scale, torch.ones_like(scale))) * 127.0)
    return torch.where(m < 0, -q, q).to(torch.int8).view(-1), scale.view(-1)


def _encode_v(v):
    v = v.view(-1, BLOCK)
    scale = v.amax(dim=1, keepdim=True)
    q = torch.round(torch.sqrt(torch.sqrt(v / torch.where(scale > 0, scale, torch.ones_like(scale)))) * 255.0)
    return torch.where(v > 0, q.clamp_min(1.0), q).to(torch.uint8).view(-1), scale.view(-1)


def _decode_m(q, scale):
    q = q.view(-1, BLOCK).float()
    u = q * (1.0 / 127.0)
    return (u * u.abs() * scale.view(-1, 1)).view(-1)


def _decode_v(q, scale):
    u = q.view(-1, BLOCK).float() * (1.0 / 255.0)
    u = u * u
    return (u * u * scale.view(-1, 1)).view(-1)


def _plain_adamw(s, case):
    h = _hyper()
    b1, b2 = h["betas"]
    s["steps"] += 1
    eight = case["bits"] == 8
    g = s["grad"].float()
    m = _decode_m(s["m"], s["m_scale"]) if eight else s["m"]
    v = _decode_v(s["v"], s["v_scale"]) if eight else s["v"]
    m = m * b1 + g * (1.0 - b1)
    v = v * b2 + (g * g) * (1.0 - b2)
    c1, c2 = 1.0 - b1 ** s["steps"], 1.0 - b2 ** s["steps"]
    p = s["param"] if s["master"] is None else s["master"]
    p[:s["decayed"]].mul_(1.0 - h["lr"] * h["weight_decay"])
    p.sub_((h["lr"] / c1) * m / (torch.sqrt(v) * (1.0 / math.sqrt(c2)) + h["eps"]))
    if s["master"] is not None:
        s["param"].copy_(p)
    if eight:
        s["m"], s["m_scale"] = _encode_m(m)
        s["v"], s["v_scale"] = _encode_v(v)
        m, v = _decode_m(s["m"], s["m_scale"]), _decode_v(s["v"], s["v_scale"])
    else:
        s["m"], s["v"] = m, v
    return _state_of(s, m, v)


def _state_of(s, m, v):
    r = {"param": s["param"], "exp_avg": m, "exp_avg_sq": v}
    if s["master"] is not None:
        r["master"] = s["master"]
    return r


# ---------------------------------------------------------------------------------------------------------------- this package

def _own_optimizer(s, case):
    from sound_event_detection_dcase2017_task4_amd import optim
    params = [torch.nn.Parameter(s["param"][at:at + n]) for at, n in zip(s["first"], s["sizes"])]
    list(map(setattr, params, itertools.repeat("grad"), (s["grad"][at:at + n] for at, n in zip(s["first"], s["sizes"]))))
    h, k = _hyper(), _decayed(case)
    groups = [{"params": params[:k]}, {"params": params[k:], "weight_decay": 0.0}]
    opt = optim.FusedAdamW([gr for gr in groups if gr["params"]], state_bits=case["bits"], **h)
    opt.load_state_dict({"step": s["steps"], "state_bits": case["bits"], "exp_avg": s["m"], "exp_avg_sq": s["v"],
                         "exp_avg_scale": s.get("m_scale"), "exp_avg_sq_scale": s.get("v_scale"), "master": s["master"]})
    return opt


def _run_own(s, case):
    if case["op"] == "adamw":
        opt = s["optimizer"]
        opt.step()
        m, v = opt.moments()
        r = {"param": s["param"], "exp_avg": m, "exp_avg_sq": v}
        if s["master"] is not None:
            r["master"] = opt.master
        return r
    from sound_event_detection_dcase2017_task4_amd import ops
    if case["op"] == "norm":
        leaves = {"gx": s["x"], "gweight": s["weight"], "gbias": s["bias"]}
        y = ops.group_norm_act(s["x"], case["groups"], s["weight"], s["bias"], eps=EPS, activation=case["act"])
    else:
        leaves = {"gx": s["x"], "gweight": s["weight"], "gbias": s["bias"]}
        if s["residual"] is not None:
            leaves["gresidual"] = s["residual"]
        y = ops.linear_act(s["x"], s["weight"], s["bias"], activation=case["act"], residual=s["residual"])
    r = {"y": y}
    if case["train"]:
        r.update(zip(leaves, torch.autograd.grad(y, list(leaves.values()), s["gy"])))
        r["y"] = y.detach()
    return r


def run(state):
    case = state["case"]
    if own:
        return _run_own(state, case)
    with torch.no_grad():
        if case["op"] == "norm":
            return _plain_norm(state, case)
        return _plain_linear(state, case) if case["op"] == "linear" else _plain_adamw(state, case)


# ---------------------------------------------------------------------------------------------------------------- what a pass needs

def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] == "norm":
        n, c = case["batch"] * case["rows"] * case["channels"], case["channels"]
        if case["train"]:                             # x, gy in; y, gx and the two parameter gradients out
            return {"bytes": 4 * n * e + 16 * c, "flops": 30 * n}
        return {"bytes": 2 * n * e + 8 * c, "flops": 10 * n}
    if case["op"] == "linear":
        M, K, N = case["m"], case["k"], case["n"]
        res = M * N if case["residual"] else 0
        if case["train"]:                             # x, W, b, residual, gy in; y, gx, gW, gb out (the residual's gradient is gy)
            return {"bytes": e * (2 * M * K + 2 * N * K + 2 * N + 2 * M * N + res), "flops": 6 * M * N * K}
        return {"bytes": e * (M * K + N * K + N + M * N + res), "flops": 2 * M * N * K}
    n = sum(_sizes(case))
    # the gradient in, the parameter in and out (16-bit ones: out, and their 32-bit copy in and out), the moments in and out;
    # 8-bit moments: codes in and out, and the values that they stand for out
    per = 3 * e if e == 4 else 2 * e + 8
    per += 16 if case["bits"] == 32 else 4 + 8
    return {"bytes": per * n, "flops": 20 * n}


# ---------------------------------------------------------------------------------------------------------------- 64 bits

def exact(case, seed):
    s = prepare({**case}, seed)
    F = torch.nn.functional
    acts = {"none": lambda z: z, "relu": F.relu, "silu": F.silu, "gelu": F.gelu}
    if case["op"] == "adamw":
        return _exact_adamw(s, case)
    leaf = {k: s[k].detach().double().requires_grad_(True) for k in ("x", "weight", "bias", "residual") if s.get(k) is not None}
    with torch.set_grad_enabled(case["train"]):
        if case["op"] == "norm":
            z = F.group_norm(leaf["x"].transpose(1, 2), case["groups"], leaf["weight"], leaf["bias"], EPS).transpose(1, 2)
            y = acts[case["act"]](z)
        else:
            y = acts[case["act"]](F.linear(leaf["x"], leaf["weight"], leaf["bias"]))
            if "residual" in leaf:
                y = y + leaf["residual"]
    out = {"y": y.detach()}
    if case["train"]:
        grads = torch.autograd.grad(y, list(leaf.values()), s["gy"].double())
        out.update({"g" + k: v for k, v in zip(leaf, grads)})
    return out


def _exact_adamw(s, case):
    """Adam with decoupled weight decay in 64 bits.  The 8-bit codes of the new moments are roundings that the last bit of a
    32-bit value decides at their borders: they have no value in 64 bits, the parameters have."""
    h = _hyper()
    (b1, b2), t = h["betas"], s["steps"] + 1
    old_m, old_v = s["m"].double(), s["v"].double()
    if case["bits"] == 8:
        per = lambda k: s[k].double().repeat_interleave(BLOCK)  # noqa: E731
        old_m = torch.sign(old_m) * torch.pow(old_m.abs() / 127.0, 2) * per("m_scale")
        old_v = torch.pow(old_v / 255.0, 4) * per("v_scale")
    g = s["grad"].double()
    m, v = torch.lerp(g, old_m, b1), torch.lerp(g.square(), old_v, b2)
    p = (s["param"] if s["master"] is None else s["master"]).double()
    rate = torch.zeros_like(p)
    rate[:s["decayed"]] = h["lr"] * h["weight_decay"]
    p = p - rate * p - h["lr"] * (m / (1.0 - b1 ** t)) / ((v / (1.0 - b2 ** t)).sqrt() + h["eps"])
    out = {"param": p, "exp_avg": m, "exp_avg_sq": v} if case["bits"] == 32 else {"param": p, "exp_avg": None, "exp_avg_sq": None}
    if s["master"] is not None:
        out["master"] = p
    return out
