"""CPU: what the channels-last layer operators refuse before any launch, and what their workspaces come to."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def L():
    from bitswap_amd import hip
    return hip.load()


def buf():
    b = (ctypes.c_char * 64)()
    return b, ctypes.c_void_p(ctypes.addressof(b))


def test_null_operands_sizes_types_and_strides_are_refused(L):
    from bitswap_amd import hip
    keep, p = buf()
    E = hip.EINVAL
    #                          x ldx  w ldw bias bt res ldr sum act  a  dt rows K  N  stream
    ok = lambda **k: L.bs_linear_act(*[k.get(n, d) for n, d in (("x", p), ("ldx", 8), ("w", p), ("ldw", 8), ("bias", None), ("bt", 0), ("res", None),      # noqa: E731
                                     ("ldr", 0), ("s", p), ("y", None), ("act", 1), ("dt", 0), ("rows", 4), ("K", 8), ("N", 8), ("ws", None), ("nb", 0), ("stream", None))])
    for bad in (dict(x=None), dict(w=None), dict(s=None), dict(ldx=7), dict(ldw=7), dict(res=p, ldr=7), dict(act=4), dict(act=-1), dict(dt=3),
                dict(dt=-1), dict(rows=-1), dict(rows=1 << 41), dict(K=0), dict(N=0), dict(bias=p, bt=1), dict(rows=100000)):
        assert ok(**bad) == E, bad
    assert ok(rows=0, x=None) == hip.OK                                     # no rows: nothing to do
    n = L.bs_linear_grad_x_workspace(0, 100000, 8, 8, 1)
    assert n > 0 and L.bs_linear_grad_x_workspace(0, 4, 8, 8, 1) == 0
    assert L.bs_linear_grad_x(None, 8, 0, p, 8, p, 0, 4, 8, 8, None, 0, None) == E
    assert L.bs_linear_grad_x(p, 7, 0, p, 8, p, 0, 4, 8, 8, None, 0, None) == E
    assert L.bs_linear_grad_x(p, 8, 0, p, 8, p, 0, 100000, 8, 8, p, n - 1, None) == E
    assert L.bs_linear_grad_x(p, 8, 0, p, 8, p, 0, 100000, 8, 8, None, n, None) == E
    assert L.bs_linear_grad_w(p, 8, 0, None, None, 8, p, 0, 4, 8, 8, None, 0, None) == E
    assert L.bs_linear_grad_w(p, 8, 0, p, None, 8, None, 0, 4, 8, 8, None, 0, None) == E
    n = L.bs_linear_grad_w_workspace(0, 100000, 8, 8, 0, 1, 1)
    assert n > 0 and L.bs_linear_grad_w(p, 8, 0, p, None, 8, p, 0, 100000, 8, 8, p, n - 1, None) == E
    assert L.bs_linear_grad_w(p, 8, 0, p, None, 8, p, 0, 100000, 8, 8, None, n, None) == E
    assert L.bs_act_grad(None, 8, None, 8, None, None, 8, 1, 0, 4, 8, p, 8, None, None, 0, None) == E           # no gradient
    assert L.bs_act_grad(None, 8, p, 8, None, None, 8, 1, 0, 4, 8, p, 8, None, None, 0, None) == E              # no sum
    assert L.bs_act_grad(p, 8, None, 8, None, None, 8, 1, 0, 4, 8, None, 8, None, None, 0, None) == E
    assert L.bs_act_grad(p, 8, None, 8, None, None, 8, 0, 0, 4, 8, p, 7, None, None, 0, None) == E           # nothing asked
    n = L.bs_act_grad_workspace(100000, 8)
    assert n > 0 and L.bs_act_grad(p, 8, None, 8, None, None, 8, 0, 0, 100000, 8, None, 8, p, p, n - 1, None) == E
    assert L.bs_group_norm_act(p, 64, 8, None, None, 0, 1e-5, 0, 0, 2, 8, 8, 3, p, None, None, 0, None) == E  # 3 groups of 8 channels
    assert L.bs_group_norm_act(p, 64, 7, None, None, 0, 1e-5, 0, 0, 2, 8, 8, 2, p, None, None, 0, None) == E
    assert L.bs_group_norm_act(p, 64, 8, p, None, 2, 1e-5, 0, 0, 2, 8, 8, 2, p, None, None, 0, None) == E     # gamma of a third type
    assert L.bs_group_norm_act(p, 64, 8, None, None, 0, -1.0, 0, 0, 2, 8, 8, 2, p, None, None, 0, None) == E
    assert L.bs_group_norm_act(p, 64, 8, None, None, 0, 1e-5, 0, 0, 2, 8000, 8, 2, p, None, None, 0, None) == E      # needs a workspace
    assert L.bs_group_norm_act_grad(p, 64, 8, p, None, 64, 8, None, None, None, 0, 0, 0, 2, 8, 8, 2, p, None, None, p, 1 << 20, None) == E
    assert L.bs_pack8(None, 8, p, p, 0, 4, 8, None) == E and L.bs_pack8(p, 7, p, p, 0, 4, 8, None) == E
    assert L.bs_pack8(p, 8, p, p, 5, 4, 8, None) == E and L.bs_unpack8(p, None, p, 0, 4, 8, None) == E
    assert L.bs_pack8(None, 8, p, p, 0, 0, 8, None) == hip.OK
    del keep


def test_workspaces(L):
    for rows in (0, 1, 63, 64, 65, 1000, 102400, 1 << 33):
        for k, n in ((1, 1), (61, 130), (2048, 2048)):
            assert 0 <= L.bs_linear_grad_w_workspace(1, rows, k, n, 0, 1, 1) < 1 << 28
            assert 0 <= L.bs_act_grad_workspace(rows, n) < 1 << 26
    assert L.bs_linear_grad_w_workspace(1, 1000, 100, 8, 1, 1, 1) == L.bs_linear_grad_w_workspace(1, 1000, 100, 8, 0, 1, 1) + 4 * 1024 * 4
    assert L.bs_linear_grad_w_workspace(1, 1000, 100, 8, 0, 0, 1) >= L.bs_linear_grad_w_workspace(1, 1000, 100, 8, 0, 1, 1) + 1000 * 104 * 2
    assert L.bs_linear_grad_w_workspace(0, 1, 8, 8, 0, 1, 1) == 0 and L.bs_linear_workspace(0, 256, 256, 256, 0) == 0
    for bad in ((3, 8, 8, 8), (1, -1, 8, 8), (1, 8, 0, 8), (1, 8, 8, 0)):
        assert L.bs_linear_grad_w_workspace(*bad, 0, 0, 0) < 0 and L.bs_linear_workspace(*bad, 1) < 0 and L.bs_linear_grad_x_workspace(*bad, 1) < 0
    assert L.bs_group_norm_workspace(0, 3, 256, 256, 32, 0) == 0
    assert L.bs_group_norm_workspace(0, 3, 1 << 20, 64, 32, 1) > 0
    assert L.bs_group_norm_workspace(0, 3, 256, 256, 33, 0) < 0


def test_tensors_off_the_gpu_are_refused():
    from bitswap_amd import hip
    x, w = torch.zeros(4, 6), torch.zeros(5, 6)
    for call in (lambda: hip.linear_act(x, w), lambda: hip.linear_act_grad(x, w, g_act=torch.zeros(4, 5)), lambda: hip.group_norm_act(x, 2),
                 lambda: hip.group_norm_act_grad(x, torch.zeros(4, 2, 2), 2, x), lambda: hip.pack8(x),
                 lambda: hip.unpack8(hip.Packed8(torch.zeros(4, 6, dtype=torch.int8), torch.zeros(4, 1, dtype=torch.int8), (4, 6), torch.float32))):
        with pytest.raises(hip.BitswapHipError):
            call()


def test_packed8_checks_its_parts():
    from bitswap_amd import hip
    codes, exps = torch.zeros(6, 40, dtype=torch.int8), torch.zeros(6, 2, dtype=torch.int8)
    p = hip.Packed8(codes, exps, (2, 3, 40), torch.bfloat16)
    assert p.shape == (2, 3, 40) and p.dtype == torch.bfloat16
    for bad in ((codes[:5], exps, (2, 3, 40)), (codes, exps[:, :1], (2, 3, 40)), (codes.int(), exps, (2, 3, 40)), (codes, exps, (2, 3, 41)),
                (codes, exps, ()), (torch.zeros(6, 80, dtype=torch.int8)[:, ::2], exps, (2, 3, 40))):
        with pytest.raises(hip.BitswapHipError):
            hip.Packed8(bad[0], bad[1], bad[2], torch.float32)
    with pytest.raises(hip.BitswapHipError):
        hip.Packed8(codes, exps, (2, 3, 40), torch.float64)


def test_rows_and_images_are_read_in_place_where_their_strides_allow():
    from bitswap_amd import hip
    x = torch.arange(2 * 3 * 4 * 10.).view(2, 3, 4, 10)
    for v, ld, rows, inplace in ((x, 10, 24, True), (x[..., 2:9], 10, 24, True), (x[:, :, ::2], 20, 12, True), (x[:, ::2], 10, 16, False),
                                 (x[0, 0, 0], 10, 1, True), (x[:, 0, 0], 120, 2, True), (x[..., ::2], 5, 24, False),
                                 (x[:1, :1, :1].expand(2, 3, 4, 10), 10, 24, False)):
        t, got, n = hip._as_rows(v, v.shape[-1], "x")
        assert (got, n) == (ld, rows) and (t.data_ptr() == v.data_ptr()) == inplace
        flat = torch.as_strided(t, (n, v.shape[-1]), (got, 1))
        assert torch.equal(flat, v.reshape(-1, v.shape[-1]))
    for v, inplace in ((x, True), (x[:, :, :, 1:7], True), (x[::2], True), (x[:, :, ::2], True), (x[:, ::2], False), (x[:, 0], True), (x[:, 0, 0], True),
                       (x.permute(0, 3, 1, 2), False), (x[:1].expand(5, 3, 4, 10), True)):
        t, ldn, ldp, n, pixels, c = hip._as_images(v, "x")
        assert (t.data_ptr() == v.data_ptr()) == inplace
        assert torch.equal(torch.as_strided(t, (n, pixels, c), (ldn, ldp, 1)), v.reshape(n, pixels, c))


def test_layers_on_the_cpu_and_the_models_option():
    """The plain path: gradients against differences; Model(npoint=0) is the reference's architecture, npoint > 0 adds parameters
    and changes no other one."""
    from bitswap_amd.layers import PointwiseResNetLayer, groups_for
    from bitswap_amd.model import Model
    assert [groups_for(c) for c in (256, 252, 254, 255, 64, 61, 16)] == [32, 28, 2, 17, 32, 1, 16]
    torch.manual_seed(3)
    for act in ("none", "elu", "silu", "gelu"):
        layer = PointwiseResNetLayer(6, hidden=5, groups=3, act=act).double()
        x = torch.randn(2, 3, 2, 6, dtype=torch.float64, requires_grad=True)
        assert torch.autograd.gradcheck(lambda *a: layer(a[0]), (x,) + tuple(layer.parameters()), atol=1e-6)
    kw = dict(xs=(1, 32, 32), nz=2, zchannels=1, nprocessing=1, resdepth=2, reswidth=12)
    torch.manual_seed(5)
    plain = Model(**kw)
    torch.manual_seed(5)
    point = Model(npoint=2, **kw)
    a, b = plain.state_dict(), point.state_dict()
    assert all(torch.equal(a[k], b[k]) for k in a)
    more = set(b) - set(a)
    assert len(more) == 4 * 2 * 6 and all(k.startswith(("point_infer.", "point_gen.")) for k in more)
    torch.manual_seed(6)
    lr, ld, le, _ = point.loss(torch.randint(0, 256, (2, 1, 32, 32)).float())
    (-lr + (le - ld).sum()).backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in point.parameters() if p.requires_grad)
    assert point.point_gen[0][1].w2.grad.abs().sum() > 0 and point.point_infer[1][0].gamma.grad.abs().sum() > 0


def test_stream_record_names_the_pointwise_layers():
    from bitswap_amd import meta
    from bitswap_amd.model import Model
    kw = dict(xs=(1, 32, 32), nz=2, zchannels=1, nprocessing=1, resdepth=2, reswidth=12)
    assert "point" not in meta.route(Model(**kw))
    r = meta.route(Model(npoint=2, **kw))
    assert r["point"] == {"layers": 2, "rev": meta.POINT_REV}
    with pytest.raises(meta.StreamMismatch):
        meta.check({"conv_route": r}, {"conv_route": meta.route(Model(**kw))})


def test_rows_wider_than_the_kernels_offsets_are_refused(L):
    from bitswap_amd import hip
    keep, p = buf()
    E, wide = hip.EINVAL, (1 << 20) + 1
    for k, n in ((wide, 8), (8, wide)):
        assert L.bs_linear_workspace(0, 4, k, n, 1) < 0 and L.bs_linear_grad_x_workspace(0, 4, k, n, 1) < 0
        assert L.bs_linear_grad_w_workspace(0, 4, k, n, 0, 1, 1) < 0
        assert L.bs_linear_act(p, k, p, k, None, 0, None, 0, p, None, 0, 0, 4, k, n, p, 1 << 40, None) == E
        assert L.bs_linear_grad_x(p, n, 0, p, k, p, 0, 4, k, n, p, 1 << 40, None) == E
        assert L.bs_linear_grad_w(p, n, 0, p, None, k, p, 0, 4, k, n, p, 1 << 40, None) == E
    assert L.bs_linear_workspace(0, 4, 1 << 20, 8, 1) >= 0
    assert L.bs_group_norm_workspace(0, 1, 8, wide, 1, 0) < 0 and L.bs_group_norm_workspace(0, 1 << 40, 8, 8, 1, 1) < 0
    assert L.bs_pack8(p, 1 << 30, p, p, 0, 1 << 40, 1 << 30, None) == E and L.bs_unpack8(p, p, p, 0, 1 << 40, 1 << 30, None) == E
    del keep


def test_act_grad_without_rows_needs_no_output(L):
    """An empty ds has no address: without rows and without db there is nothing to write, and nothing to refuse."""
    from bitswap_amd import hip
    keep, p = buf()
    assert L.bs_act_grad(p, 8, None, 8, None, None, 8, 0, 0, 0, 8, None, 8, None, None, 0, None) == hip.OK
    assert L.bs_act_grad(None, 8, None, 8, None, None, 8, 1, 0, 0, 8, None, 8, None, None, 0, None) == hip.OK
    assert L.bs_act_grad(p, 8, None, 8, None, None, 8, 0, 0, 4, 8, None, 8, None, None, 0, None) == hip.EINVAL      # rows, but nothing asked
    assert L.bs_act_grad(p, 8, None, 8, None, None, 8, 0, 3, 0, 8, None, 8, None, None, 0, None) == hip.EINVAL
    del keep


def test_calls_of_more_threads_than_a_launch_has_are_refused(L):
    """2^32 threads along an axis or more: refused on the host, before a first launch writes anything."""
    from bitswap_amd import hip
    keep, p = buf()
    E, room = hip.EINVAL, 1 << 60
    assert L.bs_pack8(p, 64, p, p, 0, 1 << 30, 64, None) == E and L.bs_pack8(p, 64, p, p, 1, 1 << 30, 64, None) == E
    assert L.bs_unpack8(p, p, p, 0, 1 << 30, 64, None) == E and L.bs_unpack8(p, p, p, 2, 1 << 30, 64, None) == E
    for dt in (0, 1, 2):
        assert L.bs_linear_act(p, 8, p, 8, None, 0, None, 0, p, None, 0, dt, 1 << 34, 8, 64, p, room, None) == E           # tiles
        assert L.bs_linear_act(p, 4097, p, 4097, None, 0, None, 0, p, None, 0, dt, 1 << 25, 4097, 8, p, room, None) == E   # rows to be copied
        assert L.bs_linear_grad_x(p, 64, 0, p, 8, p, dt, 1 << 36, 8, 64, p, room, None) == E
        assert L.bs_linear_grad_w(p, 8, 0, p, None, 4097, p, dt, 1 << 25, 4097, 8, p, room, None) == E                     # rows to be copied
        assert L.bs_linear_grad_w(p, 1 << 20, 0, p, None, 1 << 20, p, dt, 1, 1 << 20, 1 << 20, p, room, None) == E         # tiles
        assert L.bs_group_norm_act(p, 8, 8, None, None, 0, 1e-5, 0, dt, 1 << 27, 1, 8, 2, p, None, None, 0, None) == E     # images that fit
        assert L.bs_group_norm_act(p, 64000, 8, None, None, 0, 1e-5, 0, dt, 1 << 20, 8000, 8, 2, p, None, p, room, None) == E      # runs
        assert L.bs_group_norm_act(p, 64 * 3000, 64, None, None, 0, 1e-5, 0, dt, 1 << 19, 3000, 64, 64, p, None, p, room, None) == E        # groups
        assert L.bs_group_norm_act_grad(p, 8, 8, p, None, 8, 8, p, None, None, 0, 0, dt, 1 << 27, 1, 8, 2, p, None, None, p, room, None) == E
        assert L.bs_group_norm_act_grad(p, 64000, 8, p, None, 64000, 8, p, None, None, 0, 0, dt, 1 << 20, 8000, 8, 2, p, None, None, p, room, None) == E
    del keep


@pytest.mark.parametrize("version,says", [(6, "ABI version 6"), (None, "ABI version None"), (7, "lacks bs_")])
def test_a_library_of_older_sources_says_so(tmp_path, monkeypatch, version, says):
    """Of another version, or of this one but without the newer entry points: what to do, not an AttributeError."""
    import subprocess
    from bitswap_amd import hip
    src, lib = tmp_path / "old.c", tmp_path / "libold.so"
    src.write_text(f"int bs_abi_version(void) {{ return {version}; }}" if version else "int bs_nothing(void) { return 0; }")
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(lib), str(src)], check=True)
    monkeypatch.setattr(hip, "_lib", None)
    monkeypatch.setattr(hip, "lib_path", lambda: str(lib))
    with pytest.raises(hip.BitswapHipError, match=says) as e:
        hip.load()
    assert "rebuild" in str(e.value)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["none", "elu", "silu", "gelu"])
def test_linear_act_on_the_cpu_rounds_16_bits_once(act, dtype):
    """As the kernels do: float32 sums, residual and activation before the one rounding of an output.  Half a step of the type beside
    the float32 sum of 40 terms, and an activation that is at most 1.13 steep."""
    from bitswap_amd import layers
    g = torch.Generator().manual_seed(3)
    x, w, b, r = (torch.randn(sh, generator=g).to(dtype) for sh in ((50, 40), (30, 40), (30,), (50, 30)))
    s, y = layers.linear_act(x, w, b, r, act=act, want_sum=True)
    s64 = x.double() @ w.double().t() + b.double() + r.double()
    mag = x.double().abs() @ w.double().abs().t() + b.double().abs() + r.double().abs()
    y64 = {"none": lambda v: v, "elu": torch.nn.functional.elu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu}[act](s64)
    half, e = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype], 1.13 * 48 * 2.0 ** -24 * mag
    assert s.dtype == y.dtype == dtype
    assert ((s.double() - s64).abs() <= half * (s64.abs() + e) + e).all()
    assert ((y.double() - y64).abs() <= half * (y64.abs() + e) + e + 8 * 2.0 ** -24).all()
    assert torch.equal(layers.linear_act(x, w, b, r, act=act), y)


def test_linear_act_on_the_cpu_refuses_what_the_kernels_do():
    from bitswap_amd import hip, layers
    x, w = torch.zeros(4, 6), torch.zeros(5, 6)
    for bad in (dict(res=torch.zeros(1, 5)), dict(res=torch.zeros(5)), dict(res=torch.zeros(4, 1)), dict(res=torch.zeros(4, 5, dtype=torch.float64)),
                dict(bias=torch.zeros(1)), dict(bias=torch.zeros(5, dtype=torch.float64)), dict(w=torch.zeros(5, 7)), dict(w=w.half()), dict(w=w[0])):
        with pytest.raises(hip.BitswapHipError):
            layers.linear_act(**{"x": x, "w": w, **bad})
    assert layers.linear_act(x.bfloat16(), w.bfloat16(), bias=torch.zeros(5)).dtype == torch.bfloat16


def test_group_norm_on_the_cpu_without_images_or_pixels():
    """As on a HIP device: an empty result, and no gradient of the parameters; the same refusals."""
    from bitswap_amd import hip, layers
    layer = layers.PointwiseResNetLayer(6, groups=3)
    for shape in ((0, 4, 4, 6), (2, 0, 4, 6), (0, 6)):
        x = torch.zeros(shape, requires_grad=True)
        y = layer(x)
        got = torch.autograd.grad(y, [x] + list(layer.parameters()), torch.zeros(shape))
        assert y.shape == got[0].shape == torch.Size(shape) and not any(v.any() for v in got[1:])
    x = torch.zeros(2, 4, 6)
    for bad in (dict(groups=4), dict(groups=0), dict(groups=2, eps=-1.0), dict(groups=2, eps=float("nan")), dict(groups=2, x=x[0, 0])):
        with pytest.raises(hip.BitswapHipError):
            layers.group_norm_act(**{"x": x, **bad})


def test_workspaces_that_are_not_aligned_are_refused(L):
    """The kernels move 16 aligned bytes of a workspace at a time."""
    from bitswap_amd import hip
    keep = (ctypes.c_char * 128)()
    at = (ctypes.addressof(keep) + 15) & ~15
    p, E, room = ctypes.c_void_p(at), hip.EINVAL, 1 << 40
    for off in (1, 4, 8):
        ws = ctypes.c_void_p(at + off)
        for dt in (0, 1, 2):
            assert L.bs_linear_act(p, 8, p, 8, None, 0, None, 0, p, None, 0, dt, 100000, 8, 8, ws, room, None) == E
            assert L.bs_linear_grad_x(p, 8, 0, p, 8, p, dt, 100000, 8, 8, ws, room, None) == E
            assert L.bs_linear_grad_w(p, 8, 0, p, None, 8, p, dt, 100000, 8, 8, ws, room, None) == E
            assert L.bs_act_grad(p, 8, None, 8, None, None, 8, 0, dt, 100000, 8, None, 8, p, ws, room, None) == E
            assert L.bs_group_norm_act(p, 64000, 8, None, None, 0, 1e-5, 0, dt, 2, 8000, 8, 2, p, None, ws, room, None) == E
            assert L.bs_group_norm_act_grad(p, 64, 8, p, None, 64, 8, p, None, None, 0, 0, dt, 2, 8, 8, 2, p, None, None, ws, room, None) == E


def test_group_norm_on_the_cpu_refuses_parameters_as_the_kernels_do():
    from bitswap_amd import hip, layers
    x, one, half = torch.randn(2, 4, 6).bfloat16(), torch.ones(6), torch.ones(6, dtype=torch.bfloat16)
    for gamma, beta in ((torch.ones(1), None), (None, torch.zeros(2, 3)), (one.double(), None), (one, half), (None, one.half())):
        with pytest.raises(hip.BitswapHipError):
            layers.group_norm_act(x, 2, gamma, beta)
    assert torch.equal(layers.group_norm_act(x, 2, one, one), layers.group_norm_act(x, 2, half, half))
