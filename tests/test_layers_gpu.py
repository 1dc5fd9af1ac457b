"""The channels-last layer operators (hip.linear_act, group_norm_act, pack8 and the gradients) against their definitions in 64 bits.

Tolerances are bounds, not measurements: an output of type t is off by half a step of t, u_t |value| with u = 2^-24, 2^-8, 2^-11;
a float32 sum of n terms by n 2^-24 sum|terms| (the six limb products of a float32 pair are exact up to 3 2^-24 of the pair); a
value rounded to t before a further product by u_t |value| there; an activation is at most 1.13 steep and is computed to a few 2^-24
of its argument."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}     # below: steps no longer shrink
E = 2.0 ** -24


@pytest.fixture(scope="module")
def hip():
    from bitswap_amd import hip as h
    h.load()
    return h


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(shape, dtype, seed, scale=1.0):
    return (torch.randn(shape, generator=gen(seed), device="cuda") * scale).to(dtype)


def act64(s, act):
    return (lambda: s, lambda: torch.nn.functional.elu(s), lambda: torch.nn.functional.silu(s), lambda: torch.nn.functional.gelu(s))[act]()


def slope64(s, act):
    s = s.detach().clone().requires_grad_()
    return torch.autograd.grad(act64(s, act).sum(), s)[0]


def close(got, want, bound, what=""):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), (what, int(bad.sum()), float((off - bound).max()), float(off.max()))


def linear64(x, w, b, r):
    s = x.double() @ w.double().t()
    mag = x.double().abs() @ w.double().abs().t()
    for t in (b, r):
        if t is not None:
            s, mag = s + t.double(), mag + t.double().abs()
    return s, mag


def check_linear(hip, x, w, b, r, act, want_sum=True):
    s, y = hip.linear_act(x, w, b, r, act=act, want_sum=want_sum)
    s64, mag = linear64(x, w, b, r)
    u, k = U[x.dtype], x.shape[-1]
    acc = (k + 8) * E * mag
    if want_sum:
        close(s, s64, u * (s64.abs() + acc) + acc + TINY[x.dtype], "sum")
    else:
        assert s is None
    y64 = act64(s64, act)
    slack = 1.13 * acc + 16 * E * (s64.abs() + 1) * (act != 0)
    close(y, y64, u * (y64.abs() + slack) + slack + TINY[x.dtype], "act")
    return s, y


SIZES = [(1, 1, 1), (1, 1024, 40), (3, 5, 7), (33, 61, 122), (129, 64, 130), (257, 252, 505), (300, 100, 31), (64, 16, 16), (31, 33, 260),
         (520, 256, 256)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,n", SIZES)
def test_linear_act(hip, rows, k, n, dtype):
    for act in range(4):
        x, w = randn((rows, k), dtype, 1), randn((n, k), dtype, 2, k ** -0.5)
        b = randn((n,), dtype if act % 2 else torch.float32, 3) if act != 2 else None
        r = randn((rows, n), dtype, 4) if act % 2 else None
        check_linear(hip, x, w, b, r, act, want_sum=act != 3)


MANY = [(8300, 96, 130), (33000, 16, 31), (33000, 61, 5), (4200, 256, 272), (4100, 1000, 512), (33100, 8, 24), (9000, 45, 130), (5001, 48, 304)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,n", MANY)
def test_linear_act_many_rows(hip, rows, k, n, dtype):
    x, w, b, r = randn((rows, k), dtype, 1), randn((n, k), dtype, 2, k ** -0.5), randn((n,), dtype, 3), randn((rows, n), dtype, 4)
    check_linear(hip, x, w, b, r, 1)
    check_linear(hip, x, w, None, None, 3, want_sum=False)
    wide = randn((rows, k + 16), dtype, 5)
    check_linear(hip, wide[:, 8:8 + k], w, b, None, 2)                    # aligned as well as its rows are
    check_linear(hip, wide[:, 3:3 + k], w, None, r, 0)                    # not aligned


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_act_strides_and_leading_axes(hip, dtype):
    wide = randn((3, 50, 80), dtype, 1)
    w = randn((40, 90), dtype, 2)[:, 3:64]                               # a slice of a wider weight: row stride 90
    r = randn((3, 50, 47), dtype, 3)[:, :, 5:45]
    check_linear(hip, wide[:, :, 7:68], w, None, r, 1)                    # channel slice, odd offset
    check_linear(hip, wide[:, ::2, 7:68], w, None, None, 2)                # every second row
    check_linear(hip, wide[1:2, 4:5, :61], w, None, None, 3)
    flip = randn((50, 61, 3), dtype, 4).permute(2, 0, 1)                  # strided channels: copied
    check_linear(hip, flip, w, None, None, 1)
    check_linear(hip, randn((1, 61), dtype, 5).expand(37, 61), w, None, None, 1)          # the same row 37 times
    check_linear(hip, randn((61,), dtype, 6), w, None, None, 0)                            # a vector
    s, y = hip.linear_act(randn((0, 61), dtype, 7), w, act=0)
    assert s is None and y.shape == (0, 40)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k,n", [(256, 256), (61, 122), (1000, 72), (40, 520)])
def test_linear_act_row_bits_do_not_depend_on_the_number_of_rows(hip, k, n, dtype):
    rows = 17000
    x, w, b, r = randn((rows, k), dtype, 1), randn((n, k), dtype, 2, k ** -0.5), randn((n,), dtype, 3), randn((rows, n), dtype, 4)
    s, y = hip.linear_act(x, w, b, r, act=1, want_sum=True)
    for lo, hi in ((0, 1), (0, 17), (5, 133), (100, 612), (1, 2000), (16999, 17000), (3, 16500)):
        s2, y2 = hip.linear_act(x[lo:hi], w, b, r[lo:hi], act=1, want_sum=True)
        assert torch.equal(s2, s[lo:hi]) and torch.equal(y2, y[lo:hi]), (lo, hi)


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_act_not_finite(hip, dtype):
    """Infinities and NaN go where float32 arithmetic takes them, and nowhere else; the other rows keep their bits."""
    x, w = randn((70, 96), dtype, 1), randn((40, 96), dtype, 2, 0.1)
    clean = hip.linear_act(x, w, act=0)[1]
    x = x.clone()
    x[3, 5], x[17, 90], x[40, 0], x[40, 1] = float("inf"), float("nan"), float("inf"), float("-inf")
    x[66, 7] = torch.finfo(dtype).max
    y = hip.linear_act(x, w, act=0)[1]
    want = torch.stack([(x.double() * w[i].double()).sum(1) for i in range(40)], 1)
    limit = torch.finfo(dtype).max * (1 + U[dtype])
    want = torch.where(want.abs() >= limit, want.sign() * math.inf, want)
    for bad in (3, 17, 40):
        assert torch.equal(y[bad].double().nan_to_num(1e300), want[bad].nan_to_num(1e300)) or \
            torch.equal(torch.isnan(y[bad]), torch.isnan(want[bad])) and torch.equal(torch.isinf(y[bad]), torch.isinf(want[bad]))
        assert torch.equal(torch.sign(y[bad].nan_to_num(0)), torch.sign(want[bad].float().nan_to_num(0)).to(dtype))
    acc = 104 * E * (x[66].double().abs() @ w.double().abs().t())
    close(y[66], want[66], U[dtype] * want[66].abs() + 2 * acc, "largest value")
    keep = [i for i in range(70) if i not in (3, 17, 40, 66)]
    assert torch.equal(y[keep], clean[keep])


def test_linear_act_activation_limits(hip):
    """act at the ends of the range: zero, both infinities, far out."""
    v = torch.tensor([0.0, -0.0, 1e-30, -1e-30, -1e-6, -20.0, -100.0, 100.0, 3e38, -3e38, float("inf"), float("-inf"), float("nan")], device="cuda")
    one = torch.ones(1, 1, device="cuda")
    for act in range(4):
        y = hip.linear_act(v.view(-1, 1), one, act=act)[1].view(-1)
        want = act64(v.double(), act).float()
        fine = torch.isfinite(want)
        if act in (1, 0):
            assert torch.equal(torch.isfinite(y), fine) and torch.equal(torch.isnan(y), torch.isnan(want))
        close(y[:10], want[:10].double(), 16 * E * (v[:10].double().abs().clamp(max=200) + 0) + U[torch.float32] * want[:10].double().abs() + 2.0 ** -126)


def test_linear_act_offsets_beyond_31_bits(hip):
    big = torch.empty((1 << 31) + 4096, dtype=torch.bfloat16, device="cuda")
    x = torch.as_strided(big, (3, 64), ((1 << 30) + 999, 1))
    x.copy_(randn((3, 64), torch.bfloat16, 1))
    check_linear(hip, x, randn((72, 64), torch.bfloat16, 2, 0.1), None, None, 1)
    g = randn((3, 72), torch.bfloat16, 3)
    dw = hip.linear_act_grad(x, randn((72, 64), torch.bfloat16, 2, 0.1), g_act=g)[1]
    want = g.double().t() @ x.double()
    close(dw, want, U[torch.bfloat16] * want.abs() + 16 * E * (g.double().abs().t() @ x.double().abs()), "dw")


# ---- the 8-bit form ---------------------------------------------------------------------------------------------------------
def eight64(x):
    """Definition in float64, one value at a time where it matters: (codes, exps, values)."""
    rows, c = x.shape
    nb = -(-c // 32)
    v = torch.nn.functional.pad(x.double(), (0, nb * 32 - c)).view(rows, nb, 32)
    fin = torch.isfinite(v)
    top = torch.where(fin, v.abs(), torch.zeros_like(v)).amax(2)
    e = torch.full(top.shape, -126, device=x.device, dtype=torch.int64)
    for k in range(-126, 9 if x.dtype == torch.float16 else 121):
        e = torch.where(top > 127 * 2.0 ** k, torch.full_like(e, k + 1), e)
    step = torch.exp2(e.double()).unsqueeze(2)
    q = torch.where(fin, torch.round(v / step).clamp(-127, 127), torch.full_like(v, -128))
    val = torch.where(fin, q * step, torch.full_like(v, math.nan))
    return q.view(rows, -1)[:, :c].to(torch.int8), e.to(torch.int8), val.view(rows, -1)[:, :c]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,c", [(1, 1), (1, 33), (7, 32), (5, 61), (3, 4), (130, 252), (64, 256), (9, 1001)])
def test_pack8_is_the_definition(hip, rows, c, dtype):
    x = randn((rows, c), dtype, rows + c)
    x = x * torch.exp2(torch.randint(-20 if dtype == torch.float16 else -100, 5, (rows, c), generator=gen(5), device="cuda").float()).to(dtype)
    p = hip.pack8(x)
    codes, exps, values = eight64(x)
    assert torch.equal(p.codes, codes) and torch.equal(p.exps, exps)
    out = hip.unpack8(p)
    assert out.dtype == dtype and torch.equal(out.double(), values)
    assert torch.equal(hip.unpack8(hip.pack8(out)), out)               # values of the form are kept


@pytest.mark.parametrize("dtype", DTYPES)
def test_pack8_borders_zeros_and_not_finite(hip, dtype):
    big = torch.finfo(dtype).max
    x = torch.zeros((8, 64), device="cuda")
    x[1, :3] = torch.tensor([127.0, 0.5, 1.5])                            # amax on the border: step 1, ties to even
    x[2, :3] = torch.tensor([127.5, 1.0, 3.0])                            # over it: step 2
    x[3, 0], x[3, 1] = float("inf"), 3.0
    x[4, 33], x[4, 34] = float("nan"), -2.0
    x[5, :] = float("-inf")
    x[6, 0], x[6, 40] = big, -big
    x[7, :4] = torch.tensor([2.0 ** -24, -2.0 ** -24, 3 * 2.0 ** -24, 0.0])
    x = x.to(dtype)
    if dtype != torch.float16:
        x[0, :3] = torch.tensor([2.0 ** -126, 2.0 ** -127, 1.5 * 2.0 ** -126]).to(dtype)
    p = hip.pack8(x)
    codes, exps, values = eight64(x)
    assert torch.equal(p.codes, codes) and torch.equal(p.exps, exps)
    out = hip.unpack8(p).double()
    assert torch.equal(out.nan_to_num(nan=1e300), values.nan_to_num(nan=1e300))
    assert int(torch.isnan(out).sum()) == 1 + 1 + 64


def test_pack8_shapes_and_strides(hip):
    x = randn((2, 3, 5, 90), torch.float32, 1)
    for v in (x, x[:, :, :, 3:70], x[:, ::2], x.transpose(0, 1), x[0, 0, 0]):
        p = hip.pack8(v)
        assert p.shape == tuple(v.shape) and p.dtype == v.dtype
        assert torch.equal(hip.unpack8(p).double(), eight64(v.reshape(-1, v.shape[-1]))[2].view(v.shape))
    assert hip.unpack8(hip.pack8(x[:0])).shape == (0, 3, 5, 90)


# ---- gradients of the product -----------------------------------------------------------------------------------------------
def check_linear_grad(hip, x, w, s, act, gs, ga, saved8):
    """x, s float tensors; with saved8 the call gets their 8-bit form and the definition its values."""
    dt, n, k = w.dtype, w.shape[0], w.shape[1]
    xs, ss = x, s
    if saved8:
        xs, ss = hip.pack8(x), hip.pack8(s)
        x, s = hip.unpack8(xs), hip.unpack8(ss)
    dx, dw, db, dr = hip.linear_act_grad(xs, w, ss, act=act, g_sum=gs, g_act=ga, want_res=True)
    x64, s64, w64 = x.double().reshape(-1, k), s.double().reshape(-1, n), w.double()
    zero = torch.zeros_like(s64)
    a64 = ga.double().reshape(-1, n) if ga is not None else zero
    p64 = gs.double().reshape(-1, n) if gs is not None else zero
    ds = p64 + a64 * slope64(s64, act)
    u, rows = U[dt], ds.shape[0]
    # ds in float32: the slope to 16 2^-24 of (1 + |s|), then rounded to the type unless it is a gradient as it came
    made = (act != 0 and ga is not None) or (gs is not None and ga is not None)
    e32 = (16 * E * (1 + s64.abs()) * a64.abs() * (act != 0) + 2 * E * (p64.abs() + a64.abs())) * made
    eds = e32 + (u * (ds.abs() + e32) + TINY[dt]) * made
    close(dr.reshape(-1, n), ds, eds, "dres")
    close(db, ds.sum(0), e32.sum(0) + (rows + 8) * E * ds.abs().sum(0) + E * ds.sum(0).abs(), "db")
    for got, want, mag, off, terms, name in (
            (dx.reshape(-1, k), ds @ w64, ds.abs() @ w64.abs(), eds @ w64.abs(), n, "dx"),
            (dw, ds.t() @ x64, ds.t().abs() @ x64.abs(), eds.t() @ x64.abs(), rows, "dw")):
        acc = off + (terms + 8) * E * (mag + off)
        close(got, want, acc + u * (want.abs() + acc) + TINY[dt], name)
    return dx, dw, db, dr


@pytest.mark.parametrize("saved8", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,n", SIZES + [(4000, 61, 40), (2100, 300, 270)])
def test_linear_act_grad(hip, rows, k, n, dtype, saved8):
    for act in range(4):
        x, w, s = randn((rows, k), dtype, 1), randn((n, k), dtype, 2, k ** -0.5), randn((rows, n), dtype, 3)
        ga = randn((rows, n), dtype, 4, 0.1) if act != 1 or rows % 2 else randn((rows, n), dtype, 4, 0.1)
        gs = randn((rows, n), dtype, 5, 0.1) if act % 2 else None
        check_linear_grad(hip, x, w, s, act, gs, ga, saved8)
    check_linear_grad(hip, x, w, s, 1, gs, None, saved8)                  # the sum's gradient alone


@pytest.mark.parametrize("saved8", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,n", MANY)
def test_linear_act_grad_many_rows(hip, rows, k, n, dtype, saved8):
    x, w, s = randn((rows, k), dtype, 1), randn((n, k), dtype, 2, k ** -0.5), randn((rows, n), dtype, 3)
    check_linear_grad(hip, x, w, s, 2, randn((rows, n), dtype, 5, 0.1), randn((rows, n), dtype, 4, 0.1), saved8)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,n", [(70, 40, 24), (5000, 64, 144)])
def test_linear_act_grad_not_finite(hip, rows, k, n, dtype):
    """A value that was not finite when it was saved makes its column of dw NaN, and no other."""
    x, w, g = randn((rows, k), dtype, 1), randn((n, k), dtype, 2), randn((rows, n), dtype, 3)
    clean = hip.linear_act_grad(hip.pack8(x), w, g_act=g)[1]
    x = x.clone()
    x[rows // 2, 5] = float("nan")
    x[rows - 1, 33] = float("inf")
    p = hip.pack8(x)
    dw = hip.linear_act_grad(p, w, g_act=g)[1]
    hit = torch.zeros(k, dtype=torch.bool, device="cuda")
    hit[[5, 33]] = True
    assert torch.isnan(dw[:, hit]).all() and torch.isfinite(dw[:, ~hit]).all()
    other = (torch.arange(k, device="cuda") // 32 != 0) & (torch.arange(k, device="cuda") // 32 != 1)
    assert torch.equal(dw[:, other], clean[:, other])
    whole = hip.linear_act_grad(x, w, g_act=g)[1]
    want = g[:, :].double().t() @ x.double()
    assert torch.equal(torch.isnan(whole), torch.isnan(want)) and torch.equal(torch.isinf(whole), torch.isinf(want))


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_act_grad_strides(hip, dtype):
    rows, k, n = 150, 61, 43
    x, w, s = randn((rows, k + 9), dtype, 1)[:, 4:4 + k], randn((n, k + 3), dtype, 2)[:, 1:1 + k], randn((rows, n + 6), dtype, 3)[:, 5:5 + n]
    ga, gs = randn((rows, n + 2), dtype, 4)[:, 1:1 + n], randn((1, n), dtype, 5).expand(rows, n)
    check_linear_grad(hip, x, w, s, 2, gs, ga, False)
    check_linear_grad(hip, x, w, s, 0, None, ga, False)                   # nothing made: the gradient itself, strided
    check_linear_grad(hip, x, w, s, 0, gs, None, False)                   # ... or one row for all
    check_linear_grad(hip, x.view(5, 30, k) if x.is_contiguous() else x.unflatten(0, (5, 30)), w, s.unflatten(0, (5, 30)), 1,
                      None, ga.unflatten(0, (5, 30)), True)


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_act_grad_without_rows(hip, dtype):
    w = randn((6, 5), dtype, 1)
    x, s, g = (torch.empty((0, c), dtype=dtype, device="cuda") for c in (5, 6, 6))
    dx, dw, db, dr = hip.linear_act_grad(x, w, s, act=1, g_act=g, want_res=True)
    assert dx.shape == (0, 5) and dr.shape == (0, 6)
    assert torch.equal(dw, torch.zeros_like(w)) and torch.equal(db, torch.zeros(6, device="cuda"))


def test_linear_act_grad_only_what_is_asked(hip):
    x, w, s, g = randn((40, 24), torch.float32, 1), randn((16, 24), torch.float32, 2), randn((40, 16), torch.float32, 3), randn((40, 16), torch.float32, 4)
    whole = hip.linear_act_grad(x, w, s, act=1, g_act=g, want_res=True)
    for k, name in enumerate(("want_x", "want_w", "want_bias", "want_res")):
        ask = dict(want_x=False, want_w=False, want_bias=False, want_res=False)
        ask[name] = True
        got = hip.linear_act_grad(x if name == "want_w" else None, w, s, act=1, g_act=g, **ask)
        assert [v is not None for v in got] == [j == k for j in range(4)]
        assert torch.equal(got[k], whole[k])


@pytest.mark.parametrize("act", range(4))
def test_linear_act_grad_against_differences(hip, act):
    """Central differences of the 64-bit definition along random directions."""
    rows, k, n = 23, 19, 31
    x, w, b, r = (randn(sh, torch.float32, i) for i, sh in enumerate([(rows, k), (n, k), (n,), (rows, n)]))
    ga, gs = randn((rows, n), torch.float32, 7), randn((rows, n), torch.float32, 8)

    def loss(x, w, b, r):
        s = x @ w.t() + b + r
        return (ga.double() * act64(s, act) + gs.double() * s).sum()
    s = hip.linear_act(x, w, b, r, act=act, want_sum=True)[0]
    got = hip.linear_act_grad(x, w, s, act=act, g_sum=gs, g_act=ga, want_res=True)
    at = [t.double() for t in (x, w, b, r)]
    for i, d in enumerate(got):
        v = randn(at[i].shape, torch.float64, 20 + i)
        h = 1e-5
        up, down = [list(at) for _ in range(2)]
        up[i], down[i] = at[i] + h * v, at[i] - h * v
        want = (loss(*up) - loss(*down)) / (2 * h)
        have = (d.double() * v).sum()
        # gradients to about 1e-5 of their magnitude (sums of up to 31 float32 terms and s rounded), ELU's kink: second-order h
        assert abs(have - want) <= 2e-5 * (d.double().abs() * v.abs()).sum() + 1e-3 * h * v.numel()


# ---- group norm -------------------------------------------------------------------------------------------------------------
def norm64(x, groups, gamma, beta, eps):
    n, c = x.shape[0], x.shape[-1]
    v = x.double().reshape(n, -1, groups, c // groups)
    mean = v.mean((1, 3), keepdim=True)
    var = (v - mean).square().mean((1, 3), keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    h = ((v - mean) * rstd).reshape(n, -1, c)
    u = h * (gamma.double() if gamma is not None else 1) + (beta.double() if beta is not None else 0)
    return mean.view(n, groups), rstd.view(n, groups), h, u


NORMS = [(1, 1, 8, 2), (1, 1, 64, 1), (2, 16, 6, 3), (3, 49, 61, 1), (5, 64, 48, 4), (1, 256, 256, 32), (3, 289, 252, 28), (2, 1000, 64, 1),
         (2, 1024, 60, 10), (1, 2500, 24, 3), (1, 300, 1040, 2), (2, 225, 2048, 32), (7, 3, 2048, 1)]


def norm_bounds(x, mean, rstd, h, u, gamma, groups):
    """How far the statistics and u may be in float32: the mean by count 2^-24 mean|x| at worst -- the sums run over at most 32
    terms a thread, then lanes: 300 2^-24 covers every order used -- and everything behind follows from it."""
    n, c = x.shape[0], x.shape[-1]
    per = c // groups
    v = x.double().reshape(n, -1, groups, per)
    big = v.abs().amax((1, 3))
    e_mean = 64 * E * v.abs().mean((1, 3)) + 4 * E * big
    spread = 1 / rstd
    e_var = 64 * E * spread * spread + 4 * e_mean * e_mean + 8 * E * spread * big
    e_rstd = 0.5 * e_var * rstd ** 3 + 4 * E * rstd
    wide = lambda t: t.repeat_interleave(per, 1).unsqueeze(1)      # noqa: E731
    e_h = wide(e_mean * rstd + 2 * E * big * rstd) + h.abs() * wide(e_rstd / rstd) + 4 * E * h.abs()
    g = gamma.double().abs() if gamma is not None else 1.0
    return e_mean, e_rstd, e_h * g + 4 * E * (u.abs() + (h.abs() * g))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,pixels,c,groups", NORMS)
def test_group_norm_act(hip, n, pixels, c, groups, dtype):
    for act in range(4):
        x = randn((n, pixels, c), dtype, 1, 2.0) + 0.5
        gamma = randn((c,), torch.float32 if act % 2 else dtype, 2) if act != 3 else None
        beta = randn((c,), torch.float32 if act % 2 else dtype, 3) if act != 3 else None
        y, stats, p = hip.group_norm_act(x, groups, gamma, beta, eps=1e-5, act=act, want_stats=True)
        mean, rstd, h, u = norm64(x, groups, gamma, beta, 1e-5)
        em, er, eu = norm_bounds(x, mean, rstd, h, u, gamma, groups)
        assert p is None and y.shape == x.shape and y.dtype == dtype
        close(stats[:, :, 0], mean, em + E * mean.abs(), "mean")
        close(stats[:, :, 1], rstd, er + E * rstd, "rstd")
        want = act64(u, act)
        slack = 1.13 * eu + 16 * E * (u.abs() + 1) * (act != 0)
        close(y, want, slack + U[dtype] * (want.abs() + slack) + TINY[dtype], "y")


@pytest.mark.parametrize("pixels,c,groups", [(256, 64, 8), (3000, 16, 4)])
def test_group_norm_far_from_zero(hip, pixels, c, groups):
    """A mean a thousand times the spread: the variance is taken about the mean, so only the mean's own rounding is left."""
    x = randn((2, pixels, c), torch.float32, 1) + 1000.0
    y, stats, _ = hip.group_norm_act(x, groups, act=0, want_stats=True)
    mean, rstd, h, u = norm64(x, groups, None, None, 1e-5)
    em, er, eu = norm_bounds(x, mean, rstd, h, u, None, groups)
    close(y, u, eu, "y")
    assert float(((stats[:, :, 1].double() - rstd) / rstd).abs().max()) < 1e-4


@pytest.mark.parametrize("dtype", DTYPES)
def test_group_norm_strides_and_layouts(hip, dtype):
    def same(x, groups):
        a = hip.group_norm_act(x, groups, act=2, want_stats=True)
        b = hip.group_norm_act(x.contiguous(), groups, act=2, want_stats=True)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        g = randn(tuple(x.shape), dtype, 9)
        for u, v in zip(hip.group_norm_act_grad(x, a[1], groups, g, act=2), hip.group_norm_act_grad(x.contiguous(), a[1], groups, g, act=2)):
            assert torch.equal(u, v)
    x = randn((4, 8, 9, 50), dtype, 1)
    same(x[:, :, :, 3:45], 6)
    same(x[::2, :, :, 1:41], 8)
    same(x[:, ::2], 5)
    same(x[:, :, ::3], 5)
    same(x[:1].expand(3, 8, 9, 50), 10)
    nchw = randn((3, 40, 8, 8), dtype, 2)
    same(nchw.permute(0, 2, 3, 1), 8)                                            # strided channels: copied
    same(nchw.contiguous(memory_format=torch.channels_last).permute(0, 2, 3, 1), 8)
    same(randn((4, 24), dtype, 3), 3)                                            # one vector an image
    y, st, _ = hip.group_norm_act(x[:0], 5, want_stats=True)
    assert y.shape == (0, 8, 9, 50) and st.shape == (0, 5, 2)
    y, st, _ = hip.group_norm_act(x[:, :0], 5, want_stats=True)
    assert y.shape == (4, 0, 9, 50) and torch.equal(st, torch.zeros_like(st))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pixels,c,groups", [(256, 256, 32), (289, 252, 28), (2000, 64, 8), (16, 2048, 32), (1, 96, 3)])
def test_group_norm_image_bits_do_not_depend_on_how_many(hip, pixels, c, groups, dtype):
    x, g = randn((40, pixels, c), dtype, 1), randn((40, pixels, c), dtype, 2)
    y, st, _ = hip.group_norm_act(x, groups, act=1, want_stats=True)
    dx = hip.group_norm_act_grad(x, st, groups, g, act=1)[0]
    for lo, hi in ((0, 1), (3, 5), (39, 40), (7, 30)):
        y2, st2, _ = hip.group_norm_act(x[lo:hi], groups, act=1, want_stats=True)
        assert torch.equal(y2, y[lo:hi]) and torch.equal(st2, st[lo:hi])
        assert torch.equal(hip.group_norm_act_grad(x[lo:hi], st[lo:hi], groups, g[lo:hi], act=1)[0], dx[lo:hi])


@pytest.mark.parametrize("dtype", DTYPES)
def test_group_norm_not_finite_stays_in_its_group(hip, dtype):
    for pixels in (20, 2000):
        x = randn((3, pixels, 24), dtype, 1)
        clean = hip.group_norm_act(x, 4, act=1)[0]
        x[1, pixels // 2, 7] = float("inf")
        x[2, 0, 23] = float("nan")
        y = hip.group_norm_act(x, 4, act=1)[0]
        hit = torch.zeros((3, 1, 4, 6), dtype=torch.bool, device="cuda")
        hit[1, 0, 1] = hit[2, 0, 3] = True
        hit = hit.expand(3, pixels, 4, 6).reshape(3, pixels, 24)
        assert torch.isnan(y[hit]).all() and torch.equal(y[~hit], clean[~hit])


def check_norm_grad(hip, x, groups, gamma, beta, act, g, saved8):
    dt = x.dtype
    _, stats, p = hip.group_norm_act(x, groups, gamma, beta, act=act, want_stats=True, want_pack=saved8)
    xs = p if saved8 else x
    x = hip.unpack8(p) if saved8 else x
    dx, dgamma, dbeta = hip.group_norm_act_grad(xs, stats, groups, g, gamma, beta, act=act)
    n, c = x.shape[0], x.shape[-1]
    per = c // groups
    wide = lambda t: t.double().repeat_interleave(per, 1).unsqueeze(1)      # noqa: E731
    m, r = wide(stats[:, :, 0]), wide(stats[:, :, 1])
    x64, g64 = x.double().reshape(n, -1, c), g.double().reshape(n, -1, c)
    ga, be = (gamma.double() if gamma is not None else 1.0), (beta.double() if beta is not None else 0.0)
    h = (x64 - m) * r
    u = h * ga + be
    du = g64 * slope64(u, act)
    t = du * ga
    pixels = h.shape[1]
    def mean(v):      # noqa: E306
        return v.view(n, pixels, groups, per).mean((1, 3)).repeat_interleave(per, 1).unsqueeze(1)
    dx64 = r * (t - mean(t) - h * mean(t * h))
    # float32 all the way: h to 4 2^-24 of (|x| + |m|) r, the slope to 16 2^-24 (1 + |u|) plus its own change with u (at most 1.1 per
    # unit: ELU's slope jumps nowhere), sums of count terms in lanes: 64 2^-24 of the mean magnitude
    eh = 4 * E * ((x64.abs() + m.abs()) * r)
    gabs = ga.abs() if torch.is_tensor(ga) else 1.0
    eu = eh * gabs + 4 * E * (u.abs() + h.abs() * gabs)
    edu = g64.abs() * (16 * E * (1 + u.abs()) + 1.2 * eu) * (act != 0) + 2 * E * du.abs()
    et = edu * gabs + E * t.abs()
    eth = et * h.abs() + t.abs() * eh
    e_m1 = mean(et) + 64 * E * mean(t.abs())
    e_m2 = mean(eth) + 64 * E * mean((t * h).abs())
    edx = r * (et + e_m1 + h.abs() * e_m2 + eh * mean(t * h).abs() + 8 * E * (t.abs() + mean(t).abs() + (h * mean(t * h)).abs()))
    close(dx.reshape(n, -1, c), dx64, edx + U[dt] * (dx64.abs() + edx) + TINY[dt], "dx")
    cnt = 128 + n
    close(dgamma, (du * h).sum((0, 1)), (edu * h.abs() + du.abs() * eh).sum((0, 1)) + cnt * E * (du * h).abs().sum((0, 1)), "dgamma")
    close(dbeta, du.sum((0, 1)), edu.sum((0, 1)) + cnt * E * du.abs().sum((0, 1)), "dbeta")


@pytest.mark.parametrize("saved8", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,pixels,c,groups", NORMS)
def test_group_norm_act_grad(hip, n, pixels, c, groups, dtype, saved8):
    for act in range(4):
        x, g = randn((n, pixels, c), dtype, 1, 2.0) + 0.5, randn((n, pixels, c), dtype, 4, 0.1)
        gamma = randn((c,), torch.float32 if act % 2 else dtype, 2) if act != 3 else None
        beta = randn((c,), torch.float32 if act % 2 else dtype, 3) if act != 3 else None
        check_norm_grad(hip, x, groups, gamma, beta, act, g, saved8)


def test_group_norm_grad_expanded_gradient_and_only_dx(hip):
    x = randn((3, 40, 24), torch.float32, 1)
    _, st, _ = hip.group_norm_act(x, 4, act=1, want_stats=True)
    g = torch.ones(1, 1, 1, device="cuda").expand(3, 40, 24)
    a = hip.group_norm_act_grad(x, st, 4, g, act=1)
    b = hip.group_norm_act_grad(x, st, 4, g.contiguous(), act=1, want_affine=False)
    assert torch.equal(a[0], b[0]) and b[1] is None and b[2] is None
    none = hip.group_norm_act_grad(x[:0], st[:0], 4, g[:0], act=1)
    assert none[0].shape == (0, 40, 24) and not none[1].any() and not none[2].any()


@pytest.mark.parametrize("pixels", [30, 1500])
@pytest.mark.parametrize("act", range(4))
def test_group_norm_grad_against_differences(hip, act, pixels):
    n, c, groups = 2, 12, 3
    x, g = randn((n, pixels, c), torch.float32, 1), randn((n, pixels, c), torch.float32, 2)
    gamma, beta = randn((c,), torch.float32, 3), randn((c,), torch.float32, 4)

    def loss(x, gamma, beta):
        return (g.double() * act64(norm64(x, groups, gamma, beta, 1e-5)[3], act)).sum()
    _, st, _ = hip.group_norm_act(x, groups, gamma, beta, act=act, want_stats=True)
    got = hip.group_norm_act_grad(x, st, groups, g, gamma, beta, act=act)
    at = [t.double() for t in (x, gamma, beta)]
    for i, d in enumerate(got):
        v = randn(at[i].shape, torch.float64, 20 + i)
        h = 1e-5
        up, down = [list(at) for _ in range(2)]
        up[i], down[i] = at[i] + h * v, at[i] - h * v
        want = (loss(*up) - loss(*down)) / (2 * h)
        assert abs((d.double() * v).sum() - want) <= 3e-5 * (d.double().abs() * v.abs()).sum() + 1e-3 * h * x.numel()


# ---- streams, graphs, refusals ----------------------------------------------------------------------------------------------
def test_operators_on_a_side_stream_and_in_graphs(hip):
    """Captured once each and replayed in turn, with eager work between: the same bits every time, new inputs included."""
    side = torch.cuda.Stream()

    def work(x, w, b, gamma, g):
        h, st, p = hip.group_norm_act(x, 8, gamma, b, act=1, want_stats=True, want_pack=True)
        s, y = hip.linear_act(h, w, b, x, act=2, want_sum=True)
        dx, dw, db, dr = hip.linear_act_grad(h, w, hip.pack8(s), act=2, g_act=g, want_res=True)
        return (y, s, st, dw, db, dr) + hip.group_norm_act_grad(p, st, 8, dx, gamma, b, act=1)
    graphs = []
    for k in range(2):
        a = [randn((3, 900 + 600 * k, 64), torch.float32, 1 + k), randn((64, 64), torch.float32, 2, 0.1), randn((64,), torch.float32, 3),
             randn((64,), torch.float32, 4), randn((3, 900 + 600 * k, 64), torch.float32, 5)]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            work(*a)
        torch.cuda.current_stream().wait_stream(side)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = work(*a)
        graphs.append((gr, a, out))
    for turn in range(4):
        for k, (gr, a, out) in enumerate(graphs):
            a[0].copy_(randn(tuple(a[0].shape), torch.float32, 50 + 2 * turn + k))
            gr.replay()
            want = work(*a)
            torch.cuda.synchronize()
            assert all(torch.equal(u, v) for u, v in zip(out, want)), (turn, k)


def test_refusals(hip):
    x, w = randn((4, 6), torch.float32, 1), randn((5, 6), torch.float32, 2)
    Err = hip.BitswapHipError
    for bad in (lambda: hip.linear_act(x.cpu(), w), lambda: hip.linear_act(x.double(), w.double()), lambda: hip.linear_act(x, w.half()),
                lambda: hip.linear_act(x[:, :5], w), lambda: hip.linear_act(x, w, act=9), lambda: hip.linear_act(x, w, bias=x[0]),
                lambda: hip.linear_act(x, w, res=x), lambda: hip.linear_act(x, w, want_act=False), lambda: hip.linear_act(x, w[0]),
                lambda: hip.linear_act(x, w, bias=torch.zeros(5, device="cuda", dtype=torch.float64)),
                lambda: hip.linear_act_grad(x, w), lambda: hip.linear_act_grad(x, w, g_act=x),
                lambda: hip.linear_act_grad(x, w, act=1, g_act=x[:, :5]), lambda: hip.linear_act_grad(None, w, g_act=x[:, :5]),
                lambda: hip.linear_act_grad(x[:3], w, g_act=x[:, :5]), lambda: hip.linear_act_grad(x, w, g_act=x[:, :5], g_sum=x[:3, :5]),
                lambda: hip.linear_act_grad(x, w, g_act=x[:, :5].half()),
                lambda: hip.linear_act_grad(hip.pack8(x.half()), w, g_act=x[:, :5]),
                lambda: hip.group_norm_act(x, 4), lambda: hip.group_norm_act(x, 0), lambda: hip.group_norm_act(x, 2, gamma=x[0, :5]),
                lambda: hip.group_norm_act(x, 2, eps=-1.0), lambda: hip.group_norm_act(x, 2, eps=float("nan")),
                lambda: hip.group_norm_act(x[0], 2), lambda: hip.group_norm_act(x.long(), 2),
                lambda: hip.group_norm_act_grad(x, torch.zeros(4, 3, 2, device="cuda"), 2, x),
                lambda: hip.group_norm_act_grad(x[:3], torch.zeros(4, 2, 2, device="cuda"), 2, x),
                lambda: hip.group_norm_act_grad(x, torch.zeros(4, 2, 2), 2, x),
                lambda: hip.pack8(x.long()), lambda: hip.unpack8(x), lambda: hip.pack8(x[:, :0])):
        with pytest.raises(Err):
            bad()


# ---- run together, as a layer and in the model ------------------------------------------------------------------------------------
def make_layer(c, hidden, act, dtype, save8=False, seed=1):
    from bitswap_amd.layers import PointwiseResNetLayer
    torch.manual_seed(seed)
    layer = PointwiseResNetLayer(c, hidden=hidden, act=act, save8=save8)
    with torch.no_grad():
        for p in layer.parameters():
            p.add_(0.2 * torch.randn_like(p) / math.sqrt(max(1, p.shape[-1] if p.dim() > 1 else 1)))
    return layer.to("cuda", dtype)


@pytest.mark.parametrize("act", ["elu", "silu", "gelu"])
@pytest.mark.parametrize("n,c,hidden", [(3, 64, 64), (1, 61, 122), (30, 252, 96)])
def test_layer_forward(hip, n, c, hidden, act):
    """float32, every stage's bound carried through the next one."""
    layer = make_layer(c, hidden, act, torch.float32)
    x = randn((n, 16, 16, c), torch.float32, 2)
    with torch.no_grad():
        y = layer(x)
    code = {"elu": 1, "silu": 2, "gelu": 3}[act]
    p = {k: v.detach().double() for k, v in layer.named_parameters()}
    mean, rstd, h0, u = norm64(x, layer.groups, p["gamma"], p["beta"], 1e-5)
    eu = norm_bounds(x, mean, rstd, h0, u, p["gamma"], layer.groups)[2]
    h = act64(u, code)
    eh = 1.13 * eu + 16 * E * (u.abs() + 1)
    s = h @ p["w1"].t() + p["b1"]
    es = eh @ p["w1"].abs().t() + (c + 8) * E * (h.abs() @ p["w1"].abs().t() + p["b1"].abs())
    t = act64(s, code)
    et = 1.13 * es + 16 * E * (s.abs() + 1)
    want = t @ p["w2"].t() + p["b2"] + x.double().view(n, -1, c)
    mag = t.abs() @ p["w2"].abs().t() + p["b2"].abs() + x.double().abs().view(n, -1, c)
    close(y.view(n, -1, c), want, et @ p["w2"].abs().t() + (hidden + 8) * E * mag + E * want.abs())


@pytest.mark.parametrize("save8", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_gradients_are_the_operators_chained(hip, dtype, save8):
    n, c, hidden = 5, 60, 44
    layer = make_layer(c, hidden, "silu", dtype, save8)
    x, g = randn((n, 12, 10, c), dtype, 2).requires_grad_(), randn((n, 12, 10, c), dtype, 3)
    names = [k for k, _ in layer.named_parameters()]
    got = dict(zip(["x"] + names, torch.autograd.grad(layer(x), [x] + list(layer.parameters()), g)))
    with torch.no_grad():
        put = hip.pack8 if save8 else (lambda v: v)
        h, st, _ = hip.group_norm_act(x, layer.groups, layer.gamma, layer.beta, act=2, want_stats=True)
        s1, t = hip.linear_act(h, layer.w1, layer.b1, act=2, want_sum=True)
        dt, dw2, db2, dres = hip.linear_act_grad(put(t), layer.w2, g_sum=g, want_res=True)
        dh, dw1, db1, _ = hip.linear_act_grad(put(h), layer.w1, put(s1), act=2, g_act=dt)
        dx, dgamma, dbeta = hip.group_norm_act_grad(put(x.detach()), st, layer.groups, dh, layer.gamma, layer.beta, act=2)
        want = {"x": dx + dres, "gamma": dgamma.to(dtype), "beta": dbeta.to(dtype), "w1": dw1, "b1": db1.to(dtype), "w2": dw2, "b2": db2.to(dtype)}
    for k, v in want.items():
        assert got[k].dtype == dtype and torch.equal(got[k], v), k


@pytest.mark.parametrize("act", ["elu", "gelu"])
def test_layer_gradients_against_the_cpu_in_64_bits(hip, act):
    """float32: a relative error of the whole gradient of 2^-24 times the longest sum's terms (3 x 16 x 16 x 61 values a group, added
    in runs of 32 and lanes: 300) times a condition of at most 30 for such layers: 5e-4."""
    layer = make_layer(61, 40, act, torch.float32)
    x, g = randn((3, 16, 16, 61), torch.float32, 2).requires_grad_(), randn((3, 16, 16, 61), torch.float32, 3)
    got = torch.autograd.grad(layer(x), [x] + list(layer.parameters()), g)
    import copy
    ref = copy.deepcopy(layer).cpu().double()
    x64 = x.detach().cpu().double().requires_grad_()
    want = torch.autograd.grad(ref(x64), [x64] + list(ref.parameters()), g.cpu().double())
    for a, b in zip(got, want):
        assert float((a.cpu().double() - b).norm() / b.norm()) < 5e-4


def test_saved8_takes_less_memory_and_keeps_the_forward(hip):
    used = []
    for save8 in (False, True):
        layer = make_layer(256, 256, "elu", torch.float32, save8)
        x = randn((100, 16, 16, 256), torch.float32, 2).requires_grad_()
        before = torch.cuda.memory_allocated()
        y = layer(x)
        kept = torch.cuda.memory_allocated() - before - y.numel() * 4
        used.append((y.detach(), kept))
    assert torch.equal(used[0][0], used[1][0])
    # whole: x is the caller's; h, s, t of 26 MB each.  8 bits: x, h, s, t of 6.8 MB each
    assert used[1][1] < 0.55 * used[0][1]


def test_training_step_in_a_graph(hip):
    """Forward and gradients captured, replayed between eager steps of the same leaves: the same bits."""
    layer = make_layer(64, 64, "silu", torch.bfloat16, True)
    x, g = randn((4, 16, 16, 64), torch.bfloat16, 2).requires_grad_(), randn((4, 16, 16, 64), torch.bfloat16, 3)
    leaves = [x] + list(layer.parameters())

    def step():
        return torch.autograd.grad(layer(x), leaves, g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = step()
    for k in range(3):
        with torch.no_grad():
            x.copy_(randn(tuple(x.shape), torch.bfloat16, 40 + k))
        gr.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), k


def test_model_trains_with_pointwise_layers(hip):
    from bitswap_amd.model import Model
    torch.manual_seed(4)
    kw = dict(xs=(1, 32, 32), nz=2, zchannels=1, nprocessing=1, resdepth=2, reswidth=12, npoint=1)
    for save8 in (False, True):
        m = Model(save8=save8, **kw).cuda()
        lr, ld, le, _ = m.loss(torch.randint(0, 256, (2, 1, 32, 32), device="cuda").float())
        (-lr + (le - ld).sum()).backward()
        assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in m.parameters() if p.requires_grad)
        assert m.point_gen[1][0].w1.grad.abs().sum() > 0


@pytest.mark.parametrize("small", [16, 60])          # 60: run at 64 channels by the convolutions, at 60 by the pointwise layers
def test_codec_with_pointwise_layers_is_lossless_and_batch_invariant(hip, small):
    """The layers on the coding path: (mu, scale) of a chain do not depend on how many are coded together, so streams written by four
    chains at once are read one chain at a time."""
    from bitswap_amd import workload
    from bitswap_amd.codec import BitSwapCodec
    from bitswap_amd.model import Model
    base, zend, zcen = workload.build("mnist2", torch.device("cuda"), quantbits=8, small=small)
    m = Model(xs=base.xs, nz=base.nz, zchannels=base.zchannels, nprocessing=1, kernel_size=3, resdepth=2, reswidth=small, npoint=2)
    missing = m.load_state_dict(base.cpu().state_dict(), strict=False)
    assert not missing.unexpected_keys and all(k.startswith("point_") for k in missing.missing_keys)
    m = m.cuda().eval().fold().fuse()
    m.compress(True)
    z = randn((4, base.zdim_flat), torch.float32, 8)
    with torch.no_grad():
        whole = m.generate(1)(given=z)
        for b in range(4):
            one = m.generate(1)(given=z[b:b + 1])
            assert all(torch.equal(u[b:b + 1], v) for u, v in zip(whole, one))
    images = workload.synthetic_blocks(4 * 2, m.xs, seed=3).view(4, 2, -1).to(torch.int32)
    codec = BitSwapCodec(m, zend, zcen, quantbits=8, bitswap=True)
    state, _ = codec.compress(images, nwords=2000)
    words = state.to_lists()
    from bitswap_amd import hip as h
    for b in range(4):
        one = h.RansState.from_lists([words[b]], cap=state.cap)
        out = codec.decompress(one, 2)
        assert torch.equal(out.cpu()[0], images[b])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,n", [(8300, 520, 500), (8300, 517, 500), (24700, 72, 1010)])
def test_linear_act_in_the_largest_tiles(hip, rows, k, n, dtype):
    x, w, b, r = randn((rows, k), dtype, 1), randn((n, k), dtype, 2, k ** -0.5), randn((n,), dtype, 3), randn((rows, n), dtype, 4)
    check_linear(hip, x, w, b, r, 2)
    check_linear(hip, x, randn((n, k + 8), dtype, 2, k ** -0.5)[:, 8:], None, None, 1, want_sum=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k,n", [(600, 500), (72, 1010), (1030, 300)])
def test_linear_act_row_bits_through_every_tile(hip, k, n, dtype):
    """One row, a few, and as many as fill each size of tile: the same bits wherever a row lies."""
    x, w, b = randn((24700, k), dtype, 1), randn((n, k), dtype, 2, k ** -0.5), randn((n,), dtype, 3)
    whole = hip.linear_act(x, w, b, act=1)[1]
    for rows in (1, 40, 700, 2100, 4200, 9000, 17000):
        assert torch.equal(hip.linear_act(x[:rows], w, b, act=1)[1], whole[:rows]), rows
        assert torch.equal(hip.linear_act(x[-rows:], w, b, act=1)[1], whole[-rows:]), rows


@pytest.mark.parametrize("saved8", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,n", [(24000, 300, 300), (24001, 304, 260)])
def test_linear_act_grad_in_the_largest_tiles(hip, rows, k, n, dtype, saved8):
    check_linear_grad(hip, randn((rows, k), dtype, 1), randn((n, k), dtype, 2, k ** -0.5), randn((rows, n), dtype, 5), 1, randn((rows, n), dtype, 6),
                      randn((rows, n), dtype, 7), saved8)


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_act_grad_of_one_plain_gradient_in_rows_that_are_not_whole(hip, dtype):
    """No slope and one gradient: ds is the gradient, which comes back as dres itself however its rows lie."""
    for rows, k, n in ((2151, 25, 57), (40, 16, 61), (1, 8, 1)):
        x, w = randn((rows, k), dtype, 1), randn((n, k), dtype, 2)
        for g in (randn((rows, n), dtype, 3), randn((rows, n + 5), dtype, 3)[:, 2:2 + n], randn((1, n), dtype, 3).expand(rows, n)):
            dr = check_linear_grad(hip, x, w, randn((rows, n), dtype, 4), 0, g, None, False)[3]
            assert dr is g
            dx, dw, db, dr = hip.linear_act_grad(x, w, g_sum=g, want_x=False, want_bias=False)
            assert dx is None and db is None and dr is None
            close(dw, g.double().t() @ x.double(), (rows + 8 + 2 / E * U[dtype]) * E * (g.double().abs().t() @ x.double().abs()) + TINY[dtype], "dw")


@pytest.mark.parametrize("saved8", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,pixels,c,groups", [(2, 1024, 256, 8), (2, 784, 100, 5), (1, 1000, 90, 3), (2, 256, 512, 8), (9, 225, 60, 6),
                                               (2, 3, 8192, 1), (3, 1, 8192, 1), (1, 4, 8150, 1), (1, 2, 4096, 1)])
def test_group_norm_in_the_largest_workgroups(hip, n, pixels, c, groups, dtype, saved8):
    """Groups that take more than 512 threads, and as many groups as 512 threads hold, in power-of-two lanes and in others."""
    x, g = randn((n, pixels, c), dtype, 1), randn((n, pixels, c), dtype, 4)
    gamma, beta = randn((c,), torch.float32, 2), randn((c,), torch.float32, 3)
    check_norm_grad(hip, x, groups, gamma, beta, 2, g, saved8)
    y = hip.group_norm_act(x, groups, gamma, beta, act=1)[0]
    assert torch.equal(hip.group_norm_act(x[-1:], groups, gamma, beta, act=1)[0], y[-1:])
    dx = [hip.group_norm_act_grad(x[i:], hip.group_norm_act(x[i:], groups, gamma, beta, act=1, want_stats=True)[1], groups, g[i:], gamma, beta, act=1)[0]
          for i in (0, n - 1)]
    assert torch.equal(dx[0][-1:], dx[1])


# ---- the ends of the range: many groups, no rows, far and not finite arguments -----------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,pixels,c,groups", [(2, 1, 128, 128), (3, 4, 65, 65), (2, 16, 256, 256), (1, 28, 65, 65), (2, 40, 65, 65), (1, 9, 1000, 1000),
                                               (1, 3, 250, 125), (2, 2000, 66, 66)])
def test_group_norm_stats_of_many_small_groups(hip, n, pixels, c, groups, dtype):
    """One channel a group (an instance norm): a workgroup then has more groups than threads, and each has its statistics written.
    The call itself, into memory that holds NaN."""
    x = randn((n, pixels, c), dtype, 1, 2.0) + 0.5
    y, stats = torch.empty_like(x), torch.full((n, groups, 2), math.nan, device="cuda")
    L, code = hip.load(), hip._DTYPES[dtype]
    need = L.bs_group_norm_workspace(code, n, pixels, c, groups, 0)
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    rc = L.bs_group_norm_act(x.data_ptr(), pixels * c, c, None, None, 0, 1e-5, 0, code, n, pixels, c, groups, y.data_ptr(), stats.data_ptr(),
                             ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
    assert rc == hip.OK
    mean, rstd, h, u = norm64(x, groups, None, None, 1e-5)
    em, er, eu = norm_bounds(x, mean, rstd, h, u, None, groups)
    close(stats[:, :, 0], mean, em + E * mean.abs(), "mean")
    close(stats[:, :, 1], rstd, er + E * rstd, "rstd")
    close(y, u, eu + U[dtype] * (u.abs() + eu) + TINY[dtype], "y")
    for saved8 in (False, True):
        check_norm_grad(hip, x, groups, randn((c,), torch.float32, 2), randn((c,), torch.float32, 3), 2, randn((n, pixels, c), dtype, 4, 0.1), saved8)


@pytest.mark.parametrize("dtype", DTYPES)
def test_no_rows_whatever_is_asked(hip, dtype):
    """A call without rows is one, whichever gradients are asked for; parameters' gradients are zero."""
    from itertools import product
    w = randn((6, 5), dtype, 1)
    x, s, g = (torch.empty((0, c), dtype=dtype, device="cuda") for c in (5, 6, 6))
    for act, both, saved8, *ask in product((0, 1), (False, True), (False, True), *[(False, True)] * 4):
        xs, ss = (hip.pack8(x), hip.pack8(s)) if saved8 else (x, s)
        dx, dw, db, dr = hip.linear_act_grad(xs, w, ss, act=act, g_sum=g if both else None, g_act=g, want_x=ask[0], want_w=ask[1], want_bias=ask[2],
                                             want_res=ask[3])
        assert [v is not None for v in (dx, dw, db, dr)] == ask
        assert (dx is None or dx.shape == (0, 5)) and (dr is None or dr.shape == (0, 6))
        assert (dw is None or torch.equal(dw, torch.zeros_like(w))) and (db is None or torch.equal(db, torch.zeros(6, device="cuda")))


@pytest.mark.parametrize("save8", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_layers_without_rows(hip, dtype, save8):
    from bitswap_amd import layers
    w, x = randn((6, 5), dtype, 1).requires_grad_(), randn((3, 5), dtype, 2)[:0].requires_grad_()
    y = layers.linear_act(x, w, act="silu", save8=save8)
    dx, dw = torch.autograd.grad(y, [x, w], torch.empty_like(y))
    assert y.shape == (0, 6) and dx.shape == (0, 5) and torch.equal(dw, torch.zeros_like(w))
    layer = make_layer(60, 44, "elu", dtype, save8)
    x = randn((2, 4, 4, 60), dtype, 2)[:0].requires_grad_()
    y = layer(x)
    got = torch.autograd.grad(y, [x] + list(layer.parameters()), torch.empty_like(y))
    assert y.shape == got[0].shape == (0, 4, 4, 60) and not any(v.any() for v in got[1:])


@pytest.mark.parametrize("act", range(4))
@pytest.mark.parametrize("dtype", DTYPES)
def test_activations_and_slopes_at_the_ends_of_the_range(hip, dtype, act):
    """Where a value is not finite the definition's s / (1 + e^-s), s Phi(s) in IEEE arithmetic say what comes out: SiLU and GELU of
    -inf are -inf 0 = NaN, as their slopes at either infinity are.  Finite arguments, to the type's largest: values and slopes
    by their bounds -- e^s is off by 2^-24 |s| relative and at most 2^-150 from |s| = 104 on, so |s| counts up to 104."""
    inf, big = math.inf, torch.finfo(dtype).max
    ends = torch.tensor([inf, -inf, math.nan], device="cuda").to(dtype)
    one = torch.ones(1, 1, device="cuda", dtype=dtype)
    y = hip.linear_act(ends.view(-1, 1), one, act=act)[1].view(-1).float()
    want = {0: [inf, -inf, math.nan], 1: [inf, -1.0, math.nan], 2: [inf, math.nan, math.nan], 3: [inf, math.nan, math.nan]}[act]
    assert torch.equal(y.nan_to_num(12345.0, inf, -inf), torch.tensor(want, device="cuda").nan_to_num(12345.0, inf, -inf))
    slope = hip.linear_act_grad(None, one, ends.view(-1, 1), act=act, g_act=torch.ones_like(ends).view(-1, 1), want_x=False, want_w=False,
                                want_bias=False, want_res=True)[3].view(-1).float()
    if act in (0, 1):
        assert slope[:2].tolist() == ([1.0, 1.0] if act == 0 else [1.0, 0.0])
    else:
        assert torch.isnan(slope).all()
    s = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 1e-6, -1e-6, 0.5, -0.5, 12.0, -12.0, 50.0, -50.0, 88.0, -88.0, 89.0, -89.0, 104.0, -104.0, 1e4, -1e4, big, -big],
                     device="cuda").to(dtype)
    g = torch.ones_like(s)
    ds = hip.linear_act_grad(None, one, s.view(-1, 1), act=act, g_act=g.view(-1, 1), want_x=False, want_w=False, want_bias=False, want_res=True)[3].view(-1)
    want = slope64(s.double(), act)
    off = 16 * E * (1 + s.double().abs().clamp(max=104)) * (act != 0)
    close(ds, want, off + U[dtype] * (want.abs() + off) + TINY[dtype], "slope")
    y = hip.linear_act(s.view(-1, 1), one, act=act)[1].view(-1)
    want = act64(s.double(), act)
    close(y, want, off + U[dtype] * (want.abs() + off) + TINY[dtype], "value")


@pytest.mark.parametrize("saved8", [False, True])
@pytest.mark.parametrize("c,groups", [(254, 2), (255, 17)])
def test_group_norm_at_the_presets_odd_widths(hip, c, groups, saved8):
    x, g = randn((3, 256, c), torch.float32, 1), randn((3, 256, c), torch.float32, 4, 0.1)
    gamma, beta = randn((c,), torch.float32, 2), randn((c,), torch.float32, 3)
    check_norm_grad(hip, x, groups, gamma, beta, 1, g, saved8)
    y, stats, _ = hip.group_norm_act(x, groups, gamma, beta, act=1, want_stats=True)
    mean, rstd, h, u = norm64(x, groups, gamma, beta, 1e-5)
    em, er, eu = norm_bounds(x, mean, rstd, h, u, gamma, groups)
    close(stats[:, :, 0], mean, em + E * mean.abs(), "mean")
    close(stats[:, :, 1], rstd, er + E * rstd, "rstd")
    want = act64(u, 1)
    slack = 1.13 * eu + 16 * E * (u.abs() + 1)
    close(y, want, slack + E * (want.abs() + slack), "y")
    assert torch.equal(hip.group_norm_act(x[1:2], groups, gamma, beta, act=1)[0], y[1:2])


@pytest.mark.parametrize("dataset,nz", [("cifar", 4), ("mnist", 8)])
def test_preset_with_pointwise_layers_does_not_depend_on_the_batch(hip, dataset, nz):
    """A preset's width (254, run at 256 channels by the convolutions, and 61: no whole 16-byte rows): the padding comes off and
    nothing of it is left, and every chain's (mu, scale) is the same by itself as beside others."""
    from bitswap_amd.model import preset
    torch.manual_seed(11)
    m = preset(dataset, nz, npoint=1)
    with torch.no_grad():
        for k, p in m.named_parameters():
            if k.endswith((".w2", ".beta")):
                p.add_(0.1 * torch.randn(p.shape))
    m = m.cuda().eval().fold().fuse()
    m.compress(True)
    z = randn((3, m.zdim_flat), torch.float32, 8)
    width = m.point_gen[1][0].gamma.numel()
    h = randn((2, width, 16, 16), torch.float32, 9)
    with torch.no_grad():
        want = m.point_gen[1](h.permute(0, 2, 3, 1).contiguous()).permute(0, 3, 1, 2)
        padded = torch.cat([h, h.new_zeros((2, m._cp - width, 16, 16))], 1) if m._cp > width else h
        assert torch.equal(m._point_fused("point_gen", 1, padded, False), want)
        for f in (m.generate(0), m.generate(1), m.infer(1)):
            whole = f(given=z)
            assert all(torch.isfinite(u).all() for u in whole)
            for b in range(3):
                one = f(given=z[b:b + 1])
                assert all(torch.equal(u[b:b + 1] if u.shape[0] == 3 else u, v) for u, v in zip(whole, one)), b


@pytest.mark.parametrize("rows", [64, 9000])
@pytest.mark.parametrize("sx,sw", [(1e-33, 1e20), (1e-36, 1e30), (1e-36, 1.0), (1e-38, 1e37), (1e30, 1e-36), (3e-39, 1e36)])
def test_linear_act_of_tiny_float32_operands(hip, rows, sx, sw):
    """A bfloat16 limb has no bits below 2^-133, so an operand below 2^-110 loses those of its 24 that would lie there: at most 2^-134 of
    every operand, times the other one, beside the usual bound.  (k = 48 terms, and 48 of dx; dw has `rows` of them.)"""
    n, k = 40, 48
    x, w, g = randn((rows, k), torch.float32, 1, sx), randn((n, k), torch.float32, 2, sw), randn((rows, n), torch.float32, 3, sx)
    y = hip.linear_act(x, w, act=0)[1]
    dx, dw, _, _ = hip.linear_act_grad(x, w, g_act=g, act=0)
    for got, a, b, terms in ((y, x, w.t(), k), (dx, g, w, n), (dw, g.t(), x, rows)):
        a, b = a.double().contiguous(), b.double().contiguous()
        lost = 2.0 ** -134 * (a.abs().sum(1, keepdim=True) + b.abs().sum(0, keepdim=True))
        want = a @ b
        # (dw of 1e30 times 1e30: every term is beyond the type, so a float32 sum is infinite from its first term on, with that one's sign,
        # and parts of either sign add up to NaN)
        over = want.abs() > torch.finfo(torch.float32).max
        assert not torch.isfinite(got[over]).any()
        close(got[~over], want[~over], ((terms + 8) * E * (a.abs() @ b.abs()) + lost + TINY[torch.float32])[~over])
