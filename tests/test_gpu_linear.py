"""fused_linear (mimansm1_v1_amd/linear.py) against the formulas in 64 bits.

Bounds, u = 2^-24 and h = 2^-8 (half a step of bf16): a sum of K products of
bf16 values in fp32 is off by at most K u of its magnitudes; the activations'
slopes are at most 1.13 and their second derivatives at most 0.8; z is kept in
bf16 for the backward (h |z|), and dz enters the products in bf16 (h |dz|)."""
import itertools

import pytest
import torch

from mimansm1_v1_amd import linear

pytestmark = pytest.mark.gpu

FP32, BF16, F64 = torch.float32, torch.bfloat16, torch.float64
U, H = 2.0 ** -24, 2.0 ** -8
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]
TANH_C, TANH_A = (2 / torch.pi) ** 0.5, 0.044715


def act64(name, z):
    """(act, its slope, the fp32 evaluation's error) at z."""
    one = torch.ones_like(z)
    if name == "none":
        return z, one, 0 * z
    if name == "relu":
        return z.clamp(min=0), (z > 0).to(F64), 0 * z
    if name == "silu":
        s = torch.sigmoid(z)
        # exp's argument is off by 3 u of itself, then four roundings
        return z * s, s * (1 + z * (1 - s)), (z * s).abs() * (8 + 3 * z.abs()) * U * 1.1
    if name == "gelu":
        q, pdf = 0.5 * torch.erfc(z.abs() * 0.5 ** 0.5), torch.exp(-0.5 * z * z) / (2 * torch.pi) ** 0.5
        phi = torch.where(z < 0, q, 1 - q)
        # the tail's polynomial is off by 6.3e-7 of it, its evaluation by 24 u, exp's argument by 3 u of itself
        return z * phi, phi + z * pdf, z.abs() * (q * (6.3e-7 + (24 + 2 * z * z) * U) + 2 * U * phi)
    u = 2 * TANH_C * (z + TANH_A * z ** 3)
    s, du = torch.sigmoid(u), 2 * TANH_C * (1 + 3 * TANH_A * z * z)
    return z * s, s * (1 + z * du * (1 - s)), (z * s).abs() * (8 + 9 * u.abs()) * U * 1.1


def within(name, got, want, bound):
    bound = bound * 1.01 + (H * (want.abs() + bound) if got.dtype == BF16 else U * (want.abs() + bound))
    off = (got.to(F64) - want).abs() - bound
    assert got.shape == want.shape and bool(torch.isfinite(got).all()), name
    assert off.max().item() <= 0, (name, off.max().item(), want.abs().max().item())


def make(m, k, n, dev, seed, w=BF16, flipped=False, bias=None, residual=None, x=BF16):
    g = torch.Generator(dev).manual_seed(seed)
    randn = lambda *s: torch.randn(*s, device=dev, generator=g)
    wt = (randn(k, n) * k ** -0.5).to(w).t() if flipped else (randn(n, k) * k ** -0.5).to(w)
    return (randn(m, k).to(x), wt, None if bias is None else randn(n).to(bias),
            None if residual is None else randn(m, n).to(residual))


def check(act, x, w, bias=None, residual=None, out_dtype=None, grads=True):
    leaves = [t if t is None else t.detach().requires_grad_(grads) for t in (x, w, bias, residual)]
    y = linear.fused_linear(*leaves[:3], activation=act, residual=leaves[3], out_dtype=out_dtype)
    n, k = w.shape
    x2, wd = x.detach().reshape(-1, k).to(BF16).to(F64), w.detach().to(BF16).to(F64)
    m = x2.shape[0]
    z, size = x2 @ wd.t(), x2.abs() @ wd.abs().t()
    if bias is not None:
        z, size = z + bias.to(F64), size + bias.to(F64).abs()
    dz_err = (k + 1) * U * size                                  # of z
    a, slope, a_err = act64(act, z)
    want, bound = a, 1.13 * dz_err + a_err
    if residual is not None:
        r = residual.reshape(m, n).to(F64)
        want, bound = a + r, bound + U * (a.abs() + r.abs())
    within("y", y.detach().reshape(m, n), want, bound)
    assert y.dtype == (out_dtype or (BF16 if residual is None else residual.dtype))
    assert torch.equal(y, linear.fused_linear(x, w, bias, act, residual, out_dtype))      # without gradients, again
    if not grads:
        return
    g = torch.Generator(x.device).manual_seed(99)
    dy = torch.randn(y.shape, device=x.device, generator=g).to(y.dtype)
    got = dict(zip([i for i in range(4) if leaves[i] is not None],
                   torch.autograd.grad(y, [t for t in leaves if t is not None], dy)))
    d = dy.reshape(m, n).to(F64)
    dz = d * slope
    if act == "none":
        err = 0 * dz
    else:
        # z off by its fp32 error and half a step of bf16; the slope's own evaluation by 64 u and z's terms
        zoff = dz_err + H * (z.abs() + dz_err)
        err = d.abs() * (0.8 * zoff + (64 + 16 * z.abs() * (1 + z * z)) * U)
        if act == "relu":
            err = d.abs() * (z.abs() <= dz_err * 1.01)
    rounding = H * (dz.abs() + err) if (act != "none" or dy.dtype == FP32) else 0 * dz
    for i, name in enumerate(("dx", "dw", "d_bias", "d_residual")):
        if i in got:
            assert got[i].dtype == (x, w, bias, residual)[i].dtype and got[i].shape == (x, w, bias, residual)[i].shape
    e = err + rounding
    within("dx", got[0].reshape(m, k), dz @ wd, e @ wd.abs() + n * U * (dz.abs() + e) @ wd.abs())
    within("dw", got[1], dz.t() @ x2, e.t() @ x2.abs() + m * U * (dz.abs() + e).t() @ x2.abs())
    if bias is not None:
        within("d_bias", got[2], dz.sum(0), err.sum(0) + (m + 2) * U * (dz.abs() + err).sum(0))
    if residual is not None:
        assert torch.equal(got[3], dy.to(residual.dtype).reshape(residual.shape))


@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (1, 1280, 1280), (4, 128, 77), (16, 3328, 100), (15, 1290, 17), (17, 520, 40), (5, 7, 8), (64, 200, 128), (65, 129, 65),
                                   (300, 1000, 777), (130, 384, 1), (33, 1, 320), (257, 640, 250),
                                   (3, 8200, 130), (9, 264, 8300), (16, 6144, 33), (2, 31, 1001), (13, 513, 8192)])
@pytest.mark.parametrize("flipped", [False, True])
def test_odd_and_even_sizes(hip_device, m, k, n, flipped):
    for i, act in enumerate(ACTS):
        check(act, *make(m, k, n, hip_device, 10 * i + m, flipped=flipped, bias=(FP32, BF16, None)[i % 3],
                         residual=(None, BF16, FP32)[(i + m) % 3]))


@pytest.mark.parametrize("types", list(itertools.product([BF16, FP32], [BF16, FP32], [None, BF16, FP32],
                                                         [None, BF16, FP32])))
def test_types(hip_device, types):
    x, w, bias, residual = types
    for act in ("none", "silu"):
        check(act, *make(70, 256, 136, hip_device, 3, x=x, w=w, bias=bias, residual=residual))


@pytest.mark.parametrize("out_dtype", [BF16, FP32])
@pytest.mark.parametrize("residual", [None, BF16, FP32])
def test_output_type(hip_device, out_dtype, residual):
    check("gelu", *make(40, 128, 64, hip_device, 4, bias=FP32, residual=residual), out_dtype=out_dtype)


@pytest.mark.parametrize("m,k,n,flipped", [
    (4096, 1280, 1280, False), (4096, 1280, 1280, True), (2048, 3328, 1280, True), (4000, 1280, 3328, False),
    (1500, 4096, 2048, False), (16384, 256, 1280, True), (3001, 640, 3336, True), (5000, 2000, 1000, False),
    (8192, 1280, 1280, False), (2048, 1280, 1280, True), (1024, 3328, 1283, False), (2050, 1290, 1300, True),
    (16383, 640, 200, False)])
@pytest.mark.parametrize("act", ["none", "gelu"])
def test_large_tiles(hip_device, m, k, n, flipped, act):
    """256- and 320-column tiles and those of 128 rows, whole and split along k,
    inside and across the edges."""
    check(act, *make(m, k, n, hip_device, 5, flipped=flipped, bias=FP32, residual=FP32 if act == "none" else BF16))


@pytest.mark.parametrize("m,k,n", [(16384, 256, 640), (16384, 256, 512), (9000, 1280, 1280), (600, 512, 256)])
@pytest.mark.parametrize("bias", [None, BF16, FP32])
@pytest.mark.parametrize("residual", [None, BF16, FP32])
def test_fp32_output(hip_device, m, k, n, bias, residual):
    """The layout of an fp32 output's epilogue in every width of tile, with each type beside it,
    and at an odd start of each."""
    x, w, b, r = make(m, k, n, hip_device, 15, bias=bias, residual=residual)
    check("none", x, w, b, r, FP32, grads=False)
    if residual is not None:
        wide = torch.zeros(m, n + 3, dtype=residual, device=hip_device)
        wide[:, 1:n + 1] = r
        b = None if b is None else torch.cat([b[:1], b])[1:]
        assert torch.equal(linear.fused_linear(x, w, b, residual=wide[:, 1:n + 1], out_dtype=FP32),
                           linear.fused_linear(x, w, b, residual=r, out_dtype=FP32))


@pytest.mark.parametrize("m,n,k,w_type", [
    (16384, 2560, 1280, BF16), (16391, 1275, 3300, FP32), (32768, 1280, 1280, BF16), (16384, 5120, 1280, FP32),
    (16500, 8190, 1275, BF16), (32704, 2048, 1280, FP32), (32768, 1280, 2000, BF16)])
def test_weight_gradient_of_many_rows(hip_device, m, n, k, w_type):
    """Sums over so many rows that the tiles are cut along them, to two, four and
    eight parts of both widths of tile, with what lies past the last row and column."""
    g = torch.Generator(hip_device).manual_seed(m + n)
    x, dy = (torch.randn(m, c, device=hip_device, generator=g).to(BF16) for c in (k, n))
    w = torch.zeros(n, k, device=hip_device, dtype=w_type, requires_grad=True)
    y = linear.fused_linear(x, w)
    (dw,) = torch.autograd.grad(y, w, dy)
    x64, d64 = x.to(F64), dy.to(F64)
    within("dw", dw, d64.t() @ x64, m * U * (d64.abs().t() @ x64.abs()))
    (again,) = torch.autograd.grad(linear.fused_linear(x, w), w, dy)
    assert torch.equal(dw, again)


def test_views_and_strides(hip_device):
    """x, w, bias and residual as parts of larger tensors, at odd starts, transposed,
    expanded; what lies around the output's memory is not at stake: it is new."""
    dev = hip_device
    g = torch.Generator(dev).manual_seed(6)
    big = torch.randn(40, 9, 300, device=dev, generator=g).to(BF16)
    w = torch.randn(500, 700, device=dev, generator=g).to(BF16)
    row = torch.randn(96, device=dev, generator=g)
    check("none", big[:, 2:5, 3:131], w[7:103, 11:139], row[::1], row.expand(40, 3, 96))
    check("silu", big[:, 4, :200].t(), w[:64, 1:41], row[1:65], big[3, :, :200].t()[:, :1].expand(200, 64))
    check("none", big[::2, ::3, ::2], w[:150, :90].t())
    check("gelu", big[0, 0, :128], w[:33, 64:192], row[:33], row[:33].to(BF16))
    check("none", big[:, 0, :256], w[::3, :256], None, None, FP32)


def test_rows_far_apart(hip_device):
    """Operands, residual and output gradient whose rows lie further apart than the
    tiles' 32-bit offsets reach: some columns of very wide matrices."""
    dev, far = hip_device, (1 << 24) + 8
    g = torch.Generator(dev).manual_seed(11)
    store = torch.randn(21 * far, device=dev, generator=g).to(BF16)
    part = lambda rows, cols, at: store[at:].as_strided((rows, cols), (far, 1))
    for act, flipped in itertools.product(("none", "silu"), (False, True)):
        w = part(20, 64, 8192).t() if flipped else store.as_strided((64, 128), (1 << 22, 1))
        near = w.t().contiguous().t() if flipped else w.contiguous()
        x = part(20, w.shape[1], 0)
        check(act, x, w, None, part(20, 64, 4096))
        xg = x.detach().requires_grad_(True)
        dy = part(20, 64, 1024)
        y = linear.fused_linear(xg, w, activation=act)
        (got,) = torch.autograd.grad(y, xg, dy)
        (want,) = torch.autograd.grad(linear.fused_linear(xg, near, activation=act), xg, dy.contiguous())
        assert torch.equal(got, want)


def test_two_streams_at_once(hip_device):
    """Calls that share nothing but the inputs, on two streams."""
    args = [make(300, 520, 200, hip_device, 12 + i, bias=FP32, residual=FP32) for i in range(2)]
    want = [linear.fused_linear(a[0], a[1], a[2], "gelu", a[3]) for a in args]
    streams = [torch.cuda.Stream(hip_device) for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(linear.fused_linear(args[i][0], args[i][1], args[i][2], "gelu", args[i][3]))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i in range(2) for y in got[i])


def test_changed_inputs_are_noticed(hip_device):
    """The backward reads x and w as the forward saw them, or refuses."""
    x, w, _, _ = make(20, 64, 32, hip_device, 14)
    for t in (x, w):
        x.requires_grad_(True), w.requires_grad_(True)
        y = linear.fused_linear(x, w)
        with torch.no_grad():
            t.mul_(2)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


def test_special_values(hip_device):
    """Activations at infinities, zeros and magnitudes whose exponentials overflow."""
    z = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 13.2, -13.2, 50.0, -50.0, 1e4, -1e4, 1e20, -1e20, 3e38, -3e38],
                     device=hip_device).to(BF16)
    w = torch.zeros(1, 128, dtype=BF16, device=hip_device)
    w[0, 0] = 1
    x = torch.zeros(len(z), 128, dtype=BF16, device=hip_device)
    x[:, 0] = z
    for act in ACTS:
        xg = x.clone().requires_grad_(True)
        y = linear.fused_linear(xg, w, activation=act, out_dtype=FP32)
        y.sum().backward()
        a, slope, err = act64(act, z.to(F64))
        a, slope = torch.nan_to_num(a, 0.0), torch.nan_to_num(slope, 0.0)
        if act == "gelu_tanh":       # 0 * infinity in the formula's 64 bits
            big = z.to(F64).abs() > 1e4
            a, slope, err = (torch.where(big, v, t) for t, v in ((a, z.to(F64).clamp(min=0)), (slope, (z > 0).to(F64)),
                                                                 (err, 0 * a)))
        assert bool(((y[:, 0].to(F64) - a).abs() <= torch.nan_to_num(err) + U * a.abs() + 1e-37).all()), act
        # the gradient is bf16
        assert bool(((xg.grad[:, 0].to(F64) - slope).abs() <= H * slope.abs() + 1e-5).all()), act
    for bad in (float("inf"), float("nan")):
        x[0, 0] = bad
        for act in ACTS:
            got = linear.fused_linear(x, w, activation=act, out_dtype=FP32)[0, 0].item()
            assert got == bad or got != got


def test_zero_rows_and_gradients_of_some(hip_device):
    x, w, bias, residual = make(0, 64, 32, hip_device, 7, bias=FP32, residual=BF16)
    leaves = [t.requires_grad_(True) for t in (x, w, bias, residual)]
    y = linear.fused_linear(*leaves[:3], activation="silu", residual=leaves[3])
    assert y.shape == (0, 32)
    gx, gw, gb, gr = torch.autograd.grad(y, leaves, torch.ones_like(y))
    assert gx.shape == (0, 64) and not gw.any() and not gb.any() and gr.shape == (0, 32)
    x, w, bias, residual = make(50, 72, 40, hip_device, 8, bias=FP32, residual=FP32)
    every = [t.clone().requires_grad_(True) for t in (x, w, bias, residual)]
    dy = torch.randn(50, 40, device=hip_device)
    want = torch.autograd.grad(linear.fused_linear(*every[:3], activation="gelu", residual=every[3]), every, dy)
    for i in range(4):
        some = [t.clone().requires_grad_(j == i) for j, t in enumerate((x, w, bias, residual))]
        (got,) = torch.autograd.grad(linear.fused_linear(*some[:3], activation="gelu", residual=some[3]), some[i], dy)
        assert torch.equal(got, want[i])


def test_broadcast_output_gradient(hip_device):
    x, w, bias, _ = make(30, 128, 48, hip_device, 9, bias=FP32)
    x.requires_grad_(True), w.requires_grad_(True), bias.requires_grad_(True)
    linear.fused_linear(x, w, bias, out_dtype=FP32).sum().backward()
    assert torch.equal(bias.grad, torch.full((48,), 30.0, device=hip_device))
    want = x.detach().to(F64).sum(0)
    within("dw", w.grad, want.expand(48, 128), 30 * U * x.detach().to(F64).abs().sum(0).expand(48, 128))


def test_second_derivative_is_refused(hip_device):
    x, w, _, _ = make(8, 64, 16, hip_device, 10)
    x.requires_grad_(True)
    (g,) = torch.autograd.grad(linear.fused_linear(x, w, activation="silu").sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_module_and_differences(hip_device):
    """Linear keeps nn.Linear's parameters; its gradient against differences of
    its own fp32 output (central, step 2^-4 of a bf16-exact weight)."""
    torch.manual_seed(0)
    m = linear.Linear(128, 24, activation="silu", device=hip_device, dtype=BF16)
    assert m.state_dict().keys() == torch.nn.Linear(128, 24).state_dict().keys()
    x = torch.randn(16, 128, device=hip_device).to(BF16)
    r = torch.randn(16, 24, device=hip_device)
    v = torch.randn(16, 24, device=hip_device)
    m.weight.data.copy_((m.weight * 64).round() / 64)
    (m(x, r) * v).sum().backward()
    f = lambda: (m(x, r).double() * v.double()).sum().item()
    step = 2.0 ** -6
    for i, j in ((0, 0), (5, 77), (23, 127)):
        keep = m.weight[i, j].item()
        side = []
        for s in (1, -1):
            m.weight.data[i, j] = keep + s * step
            side.append(f())
        m.weight.data[i, j] = keep
        slope = (side[0] - side[1]) / (2 * step)
        # third derivative of silu at most 0.31: step^2 / 6 of sum |v x^3|; z and dz in bf16
        mag = (v[:, i].abs() * x[:, j].float().abs()).sum().item()
        cube = (v[:, i].abs() * x[:, j].float().abs() ** 3).sum().item()
        z = (x.float() @ m.weight.float().t()).abs().max().item() + 1
        bound = step ** 2 / 6 * 0.31 * cube + mag * (3 * H * 1.1 + 0.5 * H * z) + 16 * 24 * 1e-5
        assert abs(slope - m.weight.grad[i, j].item()) <= bound, (slope, m.weight.grad[i, j].item(), bound)


def test_captured_and_replayed(hip_device):
    """Forward and backward in one graph, replayed on new values between eager work."""
    for m, k, n in ((4, 1280, 1280), (300, 200, 77), (2048, 1280, 1280)):
        x, w, bias, residual = make(m, k, n, hip_device, 11, bias=FP32, residual=FP32)
        dy = torch.randn(m, n, device=hip_device)
        leaves = [t.requires_grad_(True) for t in (x, w, bias, residual)]

        def step():
            y = linear.fused_linear(*leaves[:3], activation="gelu_tanh", residual=leaves[3])
            return [y.detach(), *torch.autograd.grad(y, leaves, dy)]      # no autograd graph outlives the step

        side = torch.cuda.Stream(hip_device)
        side.wait_stream(torch.cuda.current_stream(hip_device))
        with torch.cuda.stream(side):
            step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        for _ in range(4):
            with torch.no_grad():
                for t in (*leaves, dy):
                    t.normal_()
                w.mul_(k ** -0.5)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            want = step()
            assert all(torch.equal(a, b) for a, b in zip(got, want))
            del want


def test_refusals(hip_device):
    x, w, bias, residual = make(6, 32, 16, hip_device, 12, bias=FP32, residual=BF16)
    call = linear.fused_linear
    for bad, error in [
        (lambda: call(x.half(), w), TypeError), (lambda: call(x, w.double()), TypeError),
        (lambda: call(x.cpu(), w), ValueError), (lambda: call(x, w.cpu()), ValueError),
        (lambda: call(x, w[:, :31]), ValueError), (lambda: call(x, w[0]), ValueError),
        (lambda: call(x, w, bias[:15]), ValueError), (lambda: call(x, w, bias[None]), ValueError),
        (lambda: call(x, w, residual=residual[:5]), ValueError), (lambda: call(x, w, residual=residual[0]), ValueError),
        (lambda: call(x, w, activation="tanh"), ValueError), (lambda: call(x, w, out_dtype=torch.float16), TypeError),
        (lambda: call(3.0, w), TypeError), (lambda: linear.Linear(4, 4, activation="x"), ValueError),
    ]:
        with pytest.raises(error):
            bad()


def test_sizes_past_the_documented_ones(hip_device):
    """Refused before anything is allocated: N, K and rows, of views that take no memory."""
    some = lambda rows, cols: torch.zeros(1, 1, device=hip_device, dtype=BF16).expand(rows, cols)
    for x, w in ((some(2, 8), some(4_000_001, 8)), (some(2, 4_000_001), some(8, 4_000_001)),
                 (some((1 << 28) + 1, 8), some(8, 8)), (some((1 << 32) + 5, 8), some(8, 8))):
        with pytest.raises(ValueError, match="at most"):
            linear.fused_linear(x, w)


def infinite_and_missing(rows, dev):
    """x and w whose z = x w^T has +inf, -inf and NaN in its last three rows, ones before."""
    x = torch.zeros(rows, 1280, dtype=BF16, device=dev)
    x[:, 0] = 1
    x[rows - 3:, 0] = torch.tensor([float("inf"), -float("inf"), float("nan")], device=dev)
    w = torch.zeros(1280, 1280, dtype=BF16, device=dev)
    w[:, 0] = 1
    return x, w


@pytest.mark.parametrize("rows", [3, 40, 2100])
@pytest.mark.parametrize("act", ACTS)
def test_slopes_of_infinite_and_missing_values(hip_device, act, rows):
    """dx = dy slope(z): 1 at +inf, 0 at -inf; at a NaN relu hands dy on, the others'
    slope is NaN.  The rows around them stay finite."""
    nan = float("nan")
    x, w = infinite_and_missing(rows, hip_device)
    x.requires_grad_(True)
    y = linear.fused_linear(x, w, activation=act, out_dtype=FP32)
    dy = torch.zeros_like(y)
    dy[:, 5] = 2                                     # dx is dz w: dz's one column, in dx's first
    (dx,) = torch.autograd.grad(y, x, dy)
    wants = (2.0, 2.0 if act == "none" else 0.0, 2.0 if act in ("none", "relu") else nan)
    got = dx[rows - 3:, 0].float().tolist()
    for g, want in zip(got, wants):
        assert g != g if want != want else abs(g - want) <= 1e-30, (act, got)
    assert bool(torch.isfinite(dx[:rows - 3]).all())


@pytest.mark.parametrize("rows", [3, 40, 2100])
@pytest.mark.parametrize("act", ACTS)
def test_infinite_and_missing_values(hip_device, act, rows):
    """+inf stays, -inf becomes the activations' limit 0, a NaN stays one; the rows
    around them stay finite.  gelu's tail vanishes before -20 too."""
    x, w = infinite_and_missing(rows, hip_device)
    inf, nan = float("inf"), float("nan")
    y = linear.fused_linear(x, w, activation=act, out_dtype=FP32)
    for row, want in zip(y[rows - 3:], (inf, -inf if act == "none" else 0.0, nan)):
        assert bool((row.isnan() if want != want else row == want).all()), (act, want, row[:4])
    assert bool(torch.isfinite(y[:rows - 3]).all())
    if act == "gelu":
        x[rows - 3:, 0] = torch.tensor([-20, -1e4, -3e38], device=hip_device)
        assert not linear.fused_linear(x, w, activation=act, out_dtype=FP32)[rows - 3:].any()


@pytest.mark.parametrize("flipped", [False, True])
@pytest.mark.parametrize("act,k,n", [("none", 64, 4_000_000), ("silu", 40, 3_999_999), ("none", 4_000_000, 64),
                                     ("silu", 3_999_998, 24)])
def test_widest_matrices(hip_device, act, k, n, flipped):
    """The documented limits, forward and backward, where rows lie furthest apart."""
    check(act, *make(130, k, n, hip_device, 13, flipped=flipped, bias=FP32, residual=FP32))
    torch.cuda.empty_cache()


@pytest.mark.parametrize("act,n", [("silu", 3_999_000), ("none", 3_999_000), ("none", 1000)])
def test_strides_up_to_the_bound(hip_device, act, n):
    """The C entry with fp32 rows of output and residual as far apart as it takes them,
    where a wave has 128 of them: the values of the contiguous call, nothing else written."""
    m, k, far = 256, 64, ((1 << 30) - 64) // 127
    x, w, _, residual = make(m, k, n, hip_device, 15, residual=FP32)
    want = linear.fused_linear(x, w, activation=act, residual=residual)
    apart = torch.zeros(m * far, device=hip_device).as_strided((m, far), (far, 1))
    apart[:, :n] = residual
    out = torch.full((m * far,), 7.0, device=hip_device).as_strided((m, far), (far, 1))
    code = linear.ACTIVATIONS[act]
    keep, ws, nbytes = linear.workspace(linear._product_bytes(m, n, k, linear.ROW, code), hip_device)
    linear.call("mm1_linear", hip_device, x.data_ptr(), linear.ROW, k, w.data_ptr(), linear.ROW, k, None, 0, code,
                apart.data_ptr(), 1, far, None, 0, out.data_ptr(), 1, far, ws, nbytes, m, n, k)
    assert torch.equal(out[:, :n], want)
    assert bool((out[:, n:] == 7).all())
    del apart, out
    torch.cuda.empty_cache()
