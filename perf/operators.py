"""The channels-last layer operators of bitswap_amd.hip -- linear_act, group_norm_act, pack8 / unpack8 and the gradients of the
first two -- as cases to be timed and compared: what a residual layer over the pixels of 16x16 latents (and of anything else that
is rows of channels) spends its time on, when it answers and when it trains.

Every case is one call on tensors a program has in hand.  Sizes: 16x16 latents of 256 channels (or 61 .. 252, the narrower
presets), one chain's worth up to 400 chains at once, and generic widths up to 2048.  Saved activations in 8 bits are int8 codes
with one power of two per 32 channels of a row."""
import math

import torch

own = False

ACTS = ("none", "elu", "silu", "gelu")
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
BLOCK = 32          # channels that share a power of two
EPS = 1e-5
MOST_MACS = 16384 * 2048 * 2048
MOST_VALUES = 400 * 256 * 256


def listed():
    return [
        # a single row through a wide layer: what one latent vector costs, latency only
        {"name": "linear f16 one row", "op": "linear", "rows": 1, "cin": 1024, "cout": 1024, "dtype": "f16", "act": "elu",
         "res": False, "sum": False, "pad": 0},
        # the latent of one chain (16x16 pixels): a receiver that decodes a single stream
        {"name": "linear f32 one latent", "op": "linear", "rows": 256, "cin": 256, "cout": 256, "dtype": "f32", "act": "elu",
         "res": True, "sum": False, "pad": 0},
        # 400 chains at once, the second product of a residual layer: the sum goes on, its ELU feeds the next layer
        {"name": "linear f32 400 latents", "op": "linear", "rows": 102400, "cin": 256, "cout": 256, "dtype": "f32", "act": "elu",
         "res": True, "sum": True, "pad": 0},
        # a channel slice of a wider tensor, the 252-channel preset, an odd count of rows
        {"name": "linear bf16 ragged slice", "op": "linear", "rows": 7919, "cin": 252, "cout": 505, "dtype": "bf16", "act": "silu",
         "res": True, "sum": False, "pad": 11},
        # a wide layer on many rows: bound by the matrix cores
        {"name": "linear bf16 wide", "op": "linear", "rows": 16384, "cin": 2048, "cout": 2048, "dtype": "bf16", "act": "gelu",
         "res": False, "sum": True, "pad": 0},
        # a training step on 100 latents in float32, everything saved whole
        {"name": "linear grad f32", "op": "linear_grad", "rows": 25600, "cin": 256, "cout": 256, "dtype": "f32", "act": "elu",
         "both": True, "saved8": False},
        # a training step on 256 latents in bfloat16, its input and its sums saved in 8 bits
        {"name": "linear grad bf16 saved8", "op": "linear_grad", "rows": 65536, "cin": 512, "cout": 1024, "dtype": "bf16",
         "act": "silu", "both": False, "saved8": True},
        # the normalisation in front of it: one latent, 400 latents
        {"name": "norm f32 one latent", "op": "norm", "n": 1, "pixels": 256, "channels": 256, "groups": 32, "dtype": "f32",
         "act": "elu", "save8": False},
        {"name": "norm bf16 400 latents", "op": "norm", "n": 400, "pixels": 256, "channels": 256, "groups": 32, "dtype": "bf16",
         "act": "silu", "save8": False},
        # its gradient: 100 latents in float32; odd images of the 252-channel preset with the input saved in 8 bits
        {"name": "norm grad f32", "op": "norm_grad", "n": 100, "pixels": 256, "channels": 256, "groups": 32, "dtype": "f32",
         "act": "elu", "saved8": False},
        {"name": "norm grad f16 saved8", "op": "norm_grad", "n": 37, "pixels": 289, "channels": 252, "groups": 28, "dtype": "f16",
         "act": "gelu", "saved8": True},
        # activations of 400 latents put away in 8 bits and taken out again
        {"name": "save8 f32 400 latents", "op": "save8", "rows": 102400, "channels": 256, "dtype": "f32"},
    ]


def _spread(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "linear_grad", "norm", "norm_grad", "save8"])
    dtype = rng.choice(list(DTYPES))
    if op in ("linear", "linear_grad"):
        cin, cout = _spread(rng, 16, 2048), _spread(rng, 16, 2048)
        if rng.random() < 0.5:        # half of them the round widths that layers mostly have
            cin, cout = max(16, cin // 16 * 16), max(16, cout // 16 * 16)
        rows = _spread(rng, 1, min(102400, MOST_MACS // (2 * cin * cout), MOST_VALUES // max(cin, cout)))
        case = {"op": op, "rows": rows, "cin": cin, "cout": cout, "dtype": dtype, "act": rng.choice(ACTS)}
        if op == "linear":
            case.update(res=rng.random() < 0.5, sum=rng.random() < 0.5, pad=rng.choice([0, 0, 8, 11]))
        else:
            case.update(both=rng.random() < 0.5, saved8=rng.random() < 0.5)
        return case
    if op == "save8":
        channels = _spread(rng, 16, 2048)
        return {"op": op, "rows": _spread(rng, 1, min(102400, MOST_VALUES // channels)), "channels": channels, "dtype": dtype}
    groups, per = _spread(rng, 1, 32), _spread(rng, 1, 64)
    channels = groups * per
    pixels = rng.choice([64, 225, 256, 289, 1024, _spread(rng, 1 if per >= 16 else 16, 1024)])
    n = _spread(rng, 1, max(1, min(400, MOST_VALUES // (channels * pixels))))
    case = {"op": op, "n": n, "pixels": pixels, "channels": channels, "groups": groups, "dtype": dtype, "act": rng.choice(ACTS)}
    case["save8" if op == "norm" else "saved8"] = rng.random() < 0.5
    return case


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 13)
    return g


def _features(shape, dtype, g):
    """What such a layer sees: channels of different spread and offset."""
    c = shape[-1]
    spread = torch.empty(c, device="cuda").uniform_(0.3, 1.7, generator=g)
    offset = torch.randn(c, device="cuda", generator=g) * 0.3
    return torch.randn(shape, device="cuda", generator=g).mul_(spread).add_(offset).to(dtype)


def _eight_bits(x):
    """The 8-bit form of x [rows, C]: codes int8 [rows, C] and, per 32 channels of a row, the exponent e int8 with
    value = code 2^e: the smallest e (not below -126) whose 127 2^e covers the block."""
    rows, c = x.shape
    blocks = -(-c // BLOCK)
    v = torch.nn.functional.pad(x.float(), (0, blocks * BLOCK - c)).view(rows, blocks, BLOCK)
    m, p = torch.frexp(v.abs().amax(2))                         # amax = m 2^p, m in [0.5, 1)
    e = torch.where(m > 127.0 / 128.0, p - 6, p - 7)
    e = torch.where(m == 0, torch.full_like(e, -126), e).clamp_(min=-126)
    codes = torch.round(torch.ldexp(v, -e.unsqueeze(2))).to(torch.int8).view(rows, blocks * BLOCK)[:, :c].contiguous()
    return codes, e.to(torch.int8)


def _values(codes, exps, dtype=torch.float32):
    rows, c = codes.shape
    e = exps.to(torch.int32).repeat_interleave(BLOCK, 1)[:, :c]
    return torch.ldexp(codes.to(dtype), e)


def prepare(case, seed):
    g, dt = _generator(seed), DTYPES[case["dtype"]]
    op = case["op"]
    st = {"case": case}
    if op in ("linear", "linear_grad"):
        rows, cin, cout = case["rows"], case["cin"], case["cout"]
        st["w"] = (torch.randn((cout, cin), device="cuda", generator=g) / math.sqrt(cin)).to(dt)
        if op == "linear":
            pad = case["pad"]
            wide = _features((rows, cin + pad), dt, g)
            st["x"] = wide[:, pad // 2: pad // 2 + cin]
            st["b"] = (torch.randn(cout, device="cuda", generator=g) * 0.2).to(dt)
            st["r"] = _features((rows, cout), dt, g) if case["res"] else None
        else:
            x, s = _features((rows, cin), dt, g), _features((rows, cout), dt, g)
            st["gy"] = (torch.randn((rows, cout), device="cuda", generator=g) * 0.01).to(dt)
            st["gs"] = (torch.randn((rows, cout), device="cuda", generator=g) * 0.01).to(dt) if case["both"] else None
            st["x"], st["s"] = (_eight_bits(x), _eight_bits(s)) if case["saved8"] else (x, s)
    elif op in ("norm", "norm_grad"):
        n, pixels, channels, groups = case["n"], case["pixels"], case["channels"], case["groups"]
        x = _features((n, pixels, channels), dt, g)
        st["gamma"] = torch.randn(channels, device="cuda", generator=g) * 0.3 + 1.0
        st["beta"] = torch.randn(channels, device="cuda", generator=g) * 0.3
        st["x"] = x
        if op == "norm_grad":
            st["g"] = (torch.randn((n, pixels, channels), device="cuda", generator=g) * 0.01).to(dt)
            v = x.double().view(n, pixels, groups, channels // groups)
            mean = v.mean((1, 3))
            var = (v - mean.view(n, 1, groups, 1)).square().mean((1, 3))
            st["stats"] = torch.stack([mean, 1.0 / torch.sqrt(var + EPS)], 2).float()
            if case["saved8"]:
                st["x"] = _eight_bits(x.view(n * pixels, channels))
    else:
        st["x"] = _features((case["rows"], case["channels"]), dt, g)
    return st


# ---- the plain forms --------------------------------------------------------------------------------------------------------
def _act(s, act):
    if act == "elu":
        return torch.where(s > 0, s, torch.expm1(s))
    if act == "silu":
        return s / (1 + torch.exp(-s))
    if act == "gelu":
        return 0.5 * s * (1 + torch.erf(s * math.sqrt(0.5)))
    return s


def _slope(s, act):
    if act == "elu":
        return torch.where(s > 0, torch.ones_like(s), torch.exp(s))
    if act == "silu":
        p = 1 / (1 + torch.exp(-s))
        return p * (1 + s * (1 - p))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(s * math.sqrt(0.5))) + s * torch.exp(-0.5 * s * s) * (1 / math.sqrt(2 * math.pi))
    return torch.ones_like(s)


def _whole(v):
    return _values(*v) if isinstance(v, tuple) else v.float()


def _plain(st):
    case = st["case"]
    op, dt = case["op"], DTYPES[case["dtype"]]
    if op == "linear":
        s = st["x"].float() @ st["w"].float().t() + st["b"].float()
        if st["r"] is not None:
            s = s + st["r"].float()
        return {"sum": s.to(dt) if case["sum"] else None, "act": _act(s, case["act"]).to(dt)}
    if op == "linear_grad":
        ds = st["gy"].float() * _slope(_whole(st["s"]), case["act"])
        if st["gs"] is not None:
            ds = ds + st["gs"].float()
        return {"x": (ds @ st["w"].float()).to(dt), "w": (ds.t() @ _whole(st["x"])).to(dt), "b": ds.sum(0, dtype=torch.float64).float(),
                "res": ds.to(dt)}
    if op == "save8":
        return _values(*_eight_bits(st["x"])).to(dt)
    n, pixels, channels, groups = case["n"], case["pixels"], case["channels"], case["groups"]
    per = channels // groups
    x = _whole(st["x"]).view(n, pixels, groups, per)
    gamma, beta = st["gamma"].view(groups, per), st["beta"].view(groups, per)
    if op == "norm":
        mean = x.mean((1, 3), keepdim=True)
        rstd = 1 / torch.sqrt((x - mean).square().mean((1, 3), keepdim=True) + EPS)
        y = _act((x - mean) * rstd * gamma + beta, case["act"]).to(dt).view(n, pixels, channels)
        saved = _values(*_eight_bits(st["x"].view(n * pixels, channels))).to(dt) if case["save8"] else None
        return {"y": y, "stats": torch.cat([mean, rstd], 3).view(n, groups, 2), "saved": saved}
    mean, rstd = (st["stats"][:, :, k].view(n, 1, groups, 1) for k in (0, 1))
    h = (x - mean) * rstd
    du = st["g"].float().view(n, pixels, groups, per) * _slope(h * gamma + beta, case["act"])
    t = du * gamma
    dx = rstd * (t - t.mean((1, 3), keepdim=True) - h * (t * h).mean((1, 3), keepdim=True))
    return {"x": dx.to(dt).view(n, pixels, channels), "gamma": (du * h).sum((0, 1), dtype=torch.float64).float().view(channels),
            "beta": du.sum((0, 1), dtype=torch.float64).float().view(channels)}


# ---- the framework's calls --------------------------------------------------------------------------------------------------
def _own(st):
    from bitswap_amd import hip
    case = st["case"]
    op, dt = case["op"], DTYPES[case["dtype"]]
    act = {"none": hip.ACT_NONE, "elu": hip.ACT_ELU, "silu": hip.ACT_SILU, "gelu": hip.ACT_GELU}[case["act"]] if "act" in case else None

    def saved(v, shape):
        return hip.Packed8(v[0], v[1], shape, dt) if isinstance(v, tuple) else v
    if op == "linear":
        s, y = hip.linear_act(st["x"], st["w"], st["b"], st["r"], act=act, want_sum=case["sum"])
        return {"sum": s, "act": y}
    if op == "linear_grad":
        x, s = saved(st["x"], (case["rows"], case["cin"])), saved(st["s"], (case["rows"], case["cout"]))
        dx, dw, db, dr = hip.linear_act_grad(x, st["w"], s, act=act, g_sum=st["gs"], g_act=st["gy"], want_res=True)
        return {"x": dx, "w": dw, "b": db, "res": dr}
    if op == "save8":
        return hip.unpack8(hip.pack8(st["x"]))
    if op == "norm":
        y, stats, p = hip.group_norm_act(st["x"], case["groups"], st["gamma"], st["beta"], eps=EPS, act=act, want_stats=True,
                                         want_pack=case["save8"])
        return {"y": y, "stats": stats, "saved": hip.unpack8(p).view(-1, case["channels"]) if p is not None else None}
    x = saved(st["x"], (case["n"], case["pixels"], case["channels"]))
    dx, dgamma, dbeta = hip.group_norm_act_grad(x, st["stats"], case["groups"], st["g"], st["gamma"], st["beta"], act=act)
    return {"x": dx, "gamma": dgamma, "beta": dbeta}


def run(state):
    with torch.no_grad():
        return _own(state) if own else _plain(state)


def work(case):
    op, b = case["op"], SIZE[case["dtype"]]
    if op in ("linear", "linear_grad"):
        rows, cin, cout = case["rows"], case["cin"], case["cout"]
        macs = rows * cin * cout
        if op == "linear":
            moved = rows * cin + cin * cout + cout + rows * cout * (int(case["res"]) + 1 + int(case["sum"]))
            return {"bytes": b * moved, "flops": 2 * macs}
        kept = (1 + 1 / BLOCK) if case["saved8"] else b
        moved = kept * rows * (cin + cout) + b * (2 * cin * cout + rows * cout * (2 + int(case["both"])) + rows * cin) + 4 * cout
        return {"bytes": moved, "flops": 4 * macs}
    if op == "save8":
        values = case["rows"] * case["channels"]
        return {"bytes": 2 * values * b, "flops": 4 * values}
    values = case["n"] * case["pixels"] * case["channels"]
    small = 8 * case["channels"] + 8 * case["n"] * case["groups"]
    if op == "norm":
        return {"bytes": values * b * (3 if case["save8"] else 2) + small, "flops": 10 * values}
    return {"bytes": values * (2 * b + ((1 + 1 / BLOCK) if case["saved8"] else b)) + small + 8 * case["channels"], "flops": 20 * values}


# ---- the definitions, in 64 bits --------------------------------------------------------------------------------------------
def _act64(s, act):
    return {"none": lambda: s, "elu": lambda: torch.nn.functional.elu(s), "silu": lambda: torch.nn.functional.silu(s),
            "gelu": lambda: torch.nn.functional.gelu(s)}[act]()


def _nearest64(x):
    """x [rows, C] rounded to 8 bits per value and a power of two per 32 channels, in float64: the step is the smallest power of
    two that 127 times covers the block's largest magnitude (2^-126 at least)."""
    out = torch.empty_like(x)
    for c in range(0, x.shape[1], BLOCK):
        v = x[:, c:c + BLOCK]
        top = v.abs().amax(1, keepdim=True).clamp(min=2.0 ** -140)
        step = torch.exp2(torch.floor(torch.log2(top)) - 8)
        for _ in range(4):
            step = torch.where(127 * step < top, 2 * step, step)
        step = step.clamp(min=2.0 ** -126)
        out[:, c:c + BLOCK] = torch.round(v / step) * step
    return out


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]

    def wide(v):
        return _values(v[0], v[1], torch.float64) if isinstance(v, tuple) else v.double()
    if op == "linear":
        s = torch.nn.functional.linear(st["x"].double(), st["w"].double(), st["b"].double())
        s = s if st["r"] is None else s + st["r"].double()
        return {"sum": s if case["sum"] else None, "act": _act64(s, case["act"])}
    if op == "linear_grad":
        s = wide(st["s"]).requires_grad_()
        ds, = torch.autograd.grad(_act64(s, case["act"]), s, st["gy"].double())
        ds = ds if st["gs"] is None else ds + st["gs"].double()
        return {"x": torch.mm(ds, st["w"].double()), "w": torch.mm(ds.t().contiguous(), wide(st["x"])), "b": ds.sum(0), "res": ds}
    if op == "save8":
        return _nearest64(st["x"].double())
    n, pixels, channels, groups = case["n"], case["pixels"], case["channels"], case["groups"]
    gamma, beta = st["gamma"].double(), st["beta"].double()
    if op == "norm":
        x = st["x"].double()
        v = x.view(n, pixels, groups, -1).transpose(1, 2).reshape(n, groups, -1)
        mean, var = v.mean(2), v.var(2, unbiased=False)
        rstd = torch.rsqrt(var + EPS)
        scale = rstd.repeat_interleave(channels // groups, 1) * gamma
        shift = beta - mean.repeat_interleave(channels // groups, 1) * scale
        return {"y": _act64(x * scale.unsqueeze(1) + shift.unsqueeze(1), case["act"]), "stats": torch.stack([mean, rstd], 2),
                "saved": _nearest64(x.view(n * pixels, channels)) if case["save8"] else None}
    # the gradient with the statistics as they were saved: du through autograd, the rest from the formula per channel
    x = wide(st["x"]).view(n, pixels, channels)
    per = channels // groups
    mean = st["stats"][:, :, 0].double().repeat_interleave(per, 1).unsqueeze(1)
    rstd = st["stats"][:, :, 1].double().repeat_interleave(per, 1).unsqueeze(1)
    h = (x - mean) * rstd
    u = (h * gamma + beta).requires_grad_()
    du, = torch.autograd.grad(_act64(u, case["act"]), u, st["g"].double())

    def over_group(t):          # [n, channels] sums -> their mean over the group, for every channel
        m = t.view(n, groups, per).sum(2) / (pixels * per)
        return m.repeat_interleave(per, 1).unsqueeze(1)
    one, two = du.sum(1), (du * h).sum(1)
    dx = rstd * (du * gamma - over_group(one * gamma) - h * over_group(two * gamma))
    return {"x": dx, "gamma": two.sum(0), "beta": one.sum(0)}
