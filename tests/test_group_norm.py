"""Group norm with an activation (gfd.fused.group_norm, gfd.nn.GroupNorm): the
HIP kernels against the formula in 64 bits, forward and backward, dense and
ragged; and what it refuses.

Tolerances count roundings.  An output is off by half a step of its type, and by
fp32 arithmetic before it: xhat w + b and the activation are a few tens of
roundings of 2^-24 of the largest term (exp and erf among them count some), so
48 are allowed.  Sums are fp64, or fp32 ones of a few rows that fp64 adds up."""
import pytest
import torch

DEV = "cuda"
U = 2.0 ** -24
OPS = 48 * U


def half_step(dtype):
    return torch.finfo(dtype).eps / 2 if dtype != torch.float32 else U


def act64(z, act):
    if act == "relu":
        return torch.relu(z)
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * 0.5 ** 0.5))
    return z


def reference(x, groups, w, b, eps, act, lens=None, grad=None):
    """y and, with grad, (dx, dw, db), and the magnitudes the tolerances scale with, in fp64."""
    x = x.detach().cpu().double().requires_grad_()
    C = x.shape[-1]
    wd = torch.ones(C, dtype=torch.float64) if w is None else w.detach().cpu().double()
    bd = torch.zeros(C, dtype=torch.float64) if b is None else b.detach().cpu().double()
    wd.requires_grad_()
    bd.requires_grad_()
    if lens is None:
        parts = x.reshape(x.shape[0], -1, C).unbind(0)
    else:
        parts = torch.split(x, list(lens) + [x.shape[0] - sum(lens)])[:-1]
    out, size, back = [], [], []
    for part in parts:
        t = part.reshape(part.shape[0], groups, C // groups)
        if t.numel() == 0:
            out.append(part)
            size.append(part.detach().abs())
            back.append(part.detach().abs())
            continue
        mean = t.mean((0, 2), keepdim=True)
        var = ((t - mean) ** 2).mean((0, 2), keepdim=True)
        rstd = (var + eps).rsqrt()
        xhat = ((t - mean) * rstd).reshape(part.shape)
        out.append(act64(xhat * wd + bd, act))
        size.append(((xhat * wd).abs() + bd.abs() + 1).detach())
        back.append((rstd.expand_as(t).reshape(part.shape) * (xhat.abs() + 1)).detach())
    rest = x.shape[0] - sum(lens) if lens is not None else 0
    zero = torch.zeros(rest, C, dtype=torch.float64)
    y = torch.cat([o.reshape(-1, C) for o in out] + [zero]).reshape(x.shape)
    size = torch.cat([o.reshape(-1, C) for o in size] + [zero]).reshape(x.shape)
    back = torch.cat([o.reshape(-1, C) for o in back] + [zero]).reshape(x.shape)
    if grad is None:
        return y.detach(), size
    if not y.requires_grad:                       # no row in any segment
        return y, size, torch.zeros_like(x), torch.zeros_like(wd), torch.zeros_like(bd), back
    y = y + 0.0 * (wd.sum() + bd.sum())           # gradients of 0 where no row uses them
    gx, gw, gb = torch.autograd.grad(y, (x, wd, bd), grad.detach().cpu().double(), allow_unused=True)
    return y.detach(), size, gx, gw, gb, back


def check(x, groups, w, b, act="none", eps=1e-5, lens=None, ptr=None, grad=None):
    from gfd.fused import group_norm
    xr = x.detach().requires_grad_()
    wr = w.detach().requires_grad_() if w is not None else None
    br = b.detach().requires_grad_() if b is not None else None
    y = group_norm(xr, groups, wr, br, eps, act, ptr)
    if grad is None:
        grad = torch.randn(y.shape, generator=torch.Generator().manual_seed(1)).to(x.dtype).to(DEV)
    leaves = [t for t in (xr, wr, br) if t is not None]
    grads = iter(torch.autograd.grad(y, leaves, grad))
    ry, size, rx, rw, rb, back = reference(x, groups, w, b, eps, act, lens, grad)
    assert y.dtype == x.dtype and y.shape == x.shape
    err = (y.detach().cpu().double() - ry).abs()
    assert (err <= OPS * size + half_step(x.dtype) * ry.abs() + torch.finfo(x.dtype).tiny).all(), \
        err.max().item()
    # dx: w dz, its mean and xhat times a mean, each at most max |w dz| over the tensor;
    # |act'| <= 1.13, and act' itself moves by at most |act''| <= 1 times z's error (not relu's)
    wmax = 1.0 if w is None else w.abs().max().item()
    scale = 1.2 * wmax * grad.abs().max().item() * (1 + size.max().item() if act in ("silu", "gelu") else 1)
    gx = next(grads)
    err = (gx.cpu().double() - rx).abs()
    assert gx.dtype == x.dtype
    assert (err <= OPS * scale * 3 * back + half_step(x.dtype) * rx.abs() + torch.finfo(x.dtype).tiny).all(), \
        err.max().item()
    rows = x.numel() // x.shape[-1]
    for ours, ref, most in ((w, rw, size.max().item() / max(min(wmax, 1), 1e-2)), (b, rb, 1.0)):
        if ours is None:
            continue
        g = next(grads)
        assert g.dtype == ours.dtype
        bound = OPS * rows * scale * most + half_step(ours.dtype) * ref.abs()
        assert ((g.cpu().double() - ref).abs() <= bound).all()
    return y


def data(shape, dtype, seed=0, level=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * 1.5 + level).to(dtype).to(DEV)


def affine(C, dtype, seed=2):
    g = torch.Generator().manual_seed(seed)
    return ((1 + 0.2 * torch.randn(C, generator=g)).to(dtype).to(DEV),
            (0.2 * torch.randn(C, generator=g)).to(dtype).to(DEV))


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_rows(dtype, act):
    check(data((300, 64), dtype), 8, *affine(64, torch.float32), act=act)


@pytest.mark.gpu
@pytest.mark.parametrize("C,groups", [(1, 1), (3, 1), (3, 3), (64, 64), (64, 1), (66, 2), (83 * 2, 2),
                                      (165, 5), (24, 3), (96, 8), (1024, 32), (2048, 1), (2047, 1), (1155, 33)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_channels(C, groups, dtype):
    check(data((17, C), dtype), groups, *affine(C, dtype), act="silu")
    check(data((2, 70, C), dtype), groups, *affine(C, dtype), act="silu")


@pytest.mark.gpu
@pytest.mark.parametrize("B,L", [(1, 1), (1, 2), (3, 31), (5, 33), (1, 1000), (2, 4097), (1030, 3), (1025, 65),
                                 (4100, 9), (20, 300)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_dense_lengths(B, L, dtype):
    check(data((B, L, 24), dtype), 4, *affine(24, torch.float32), act="gelu")


@pytest.mark.gpu
@pytest.mark.parametrize("lens,behind", [
    ([5], 0), ([0], 3), ([], 4), ([1, 0, 0, 1, 7], 0), ([0, 64, 32, 33, 0], 2), ([31, 1, 32, 1, 33, 100, 0, 500], 1),
    ([700], 0), ([3] * 300, 5), ([40] * 50 + [0] * 70 + [1], 0),
    ([64, 0, 33, 96, 0, 0, 31, 32] + [1] * 60 + [1000], 3)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_ragged(lens, behind, dtype):
    n = sum(lens) + behind
    ptr = torch.tensor([0] + lens).cumsum(0).to(DEV)
    check(data((n, 32), dtype), 4, *affine(32, torch.float32), act="relu", lens=lens, ptr=ptr)


@pytest.mark.gpu
def test_ragged_with_rows_in_front():
    from gfd.fused import group_norm
    x = data((50, 16), torch.float32)
    y = group_norm(x, 2, ptr=torch.tensor([7, 20, 45], device=DEV))
    inner = group_norm(x[7:45], 2, ptr=torch.tensor([0, 13, 38], device=DEV))
    assert torch.equal(y[7:45], inner)
    assert not y[:7].any() and not y[45:].any()


@pytest.mark.gpu
def test_bad_offsets_stay_inside():
    """Offsets out of range or out of order give wrong numbers, never an access outside of the
    rows: they are clamped to them."""
    from gfd.fused import group_norm
    x = data((90, 16), torch.float32).requires_grad_()
    for at in ([-5, 40, 1000], [60, 10, 90, 3]):
        y = group_norm(x, 2, ptr=torch.tensor(at, device=DEV))
        torch.autograd.grad(y.sum(), x)
        torch.cuda.synchronize()
        assert y.shape == x.shape


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides(dtype):
    base = data((40, 6, 200), dtype)
    w, b = affine(64, torch.float32)
    check(base[:, :, 8:72], 8, w, b, act="silu")              # strided rows, aligned
    check(base[:, :, 3:67], 8, w, b, act="silu")              # an odd offset
    check(base[:, 2, 8:72], 8, w, b, act="silu")              # [N, C] with a row pitch
    check(base.transpose(0, 1)[:, :, :64], 8, w, b, act="silu")
    check(base[:, :64, :].transpose(1, 2)[:, :, :6], 3, *affine(6, torch.float32), act="none")   # channels apart
    check(base[:1, :, :64].expand(4, 6, 64), 8, w, b)         # the same rows for every sample
    g = torch.ones((), device=DEV, dtype=dtype).expand(40, 6, 64)
    check(base[:, :, :64], 8, w, b, act="relu", grad=g)       # the gradient of a sum


@pytest.mark.gpu
def test_four_dimensions_and_module_match_torch():
    from gfd.nn import GroupNorm
    m = GroupNorm(4, 32, act="relu").to(DEV)
    ref = torch.nn.GroupNorm(4, 32)
    with torch.no_grad():
        m.weight.normal_(1, 0.2)
        m.bias.normal_(0, 0.2)
    ref.load_state_dict({k: v.cpu() for k, v in m.state_dict().items()}, strict=True)
    x = data((3, 5, 7, 32), torch.float32)
    want = torch.relu(ref.double()(x.cpu().double().permute(0, 3, 1, 2))).permute(0, 2, 3, 1)
    assert (m(x).cpu().double() - want).abs().max() <= OPS * (want.abs().max() + 2)
    assert "act=relu" in repr(m)


@pytest.mark.gpu
def test_large_mean_keeps_its_digits():
    """A level 10^5 times the spread: fp32 sums of squares would lose the variance wholly."""
    x = torch.randn((64, 32), generator=torch.Generator().manual_seed(3)).to(DEV) + 1e5
    check(x, 4, *affine(32, torch.float32), act="none")


@pytest.mark.gpu
def test_constant_rows_and_zero_eps():
    from gfd.fused import group_norm
    y = group_norm(torch.full((5, 8), 3.0, device=DEV), 2, bias=torch.full((8,), 0.5, device=DEV))
    assert torch.equal(y, torch.full_like(y, 0.5))


@pytest.mark.gpu
def test_no_rows():
    from gfd.fused import group_norm
    w, b = affine(8, torch.float32)
    for shape in ((0, 8), (0, 4, 8), (4, 0, 8)):
        x = torch.empty(shape, device=DEV, requires_grad=True)
        wr = w.detach().requires_grad_()
        y = group_norm(x, 2, wr, b)
        gx, gw = torch.autograd.grad(y.sum(), (x, wr))
        assert y.shape == gx.shape == x.shape and not gw.any()


@pytest.mark.gpu
def test_nan_stays_in_its_segment():
    from gfd.fused import group_norm
    x = data((30, 16), torch.float32)
    x[4, 3] = float("nan")
    y = group_norm(x, 2, act="relu", ptr=torch.tensor([0, 10, 30], device=DEV))
    assert y[:10, :8].isnan().all() and y[:10, 8:].isfinite().all() and y[10:].isfinite().all()


@pytest.mark.gpu
def test_relu_side_of_tiny_values():
    """The gradient passes exactly where the output is not 0, and a z of exactly 0 passes none."""
    from gfd.fused import group_norm
    x = data((20000, 64), torch.float32).requires_grad_()
    y = group_norm(x, 8, act="relu")
    ry = reference(x, 8, None, None, 1e-5, "relu")[0]
    assert torch.equal(y.detach().cpu() > 0, ry > 0)


@pytest.mark.gpu
def test_gradient_against_differences():
    from gfd.fused import group_norm
    x = data((6, 9, 8), torch.float32)
    w, b = affine(8, torch.float32)
    g = data((6, 9, 8), torch.float32, seed=5)
    d = data((6, 9, 8), torch.float32, seed=6)
    for act in ("none", "silu", "gelu"):
        xr = x.clone().requires_grad_()
        gx, = torch.autograd.grad(group_norm(xr, 2, w, b, act=act), xr, g)
        h = 2.0 ** -7
        plus, minus = (group_norm(x + s * h * d, 2, w, b, act=act).double() for s in (1, -1))
        numeric = ((plus - minus) * g.double()).sum().item() / (2 * h)
        # third derivatives times h^2 / 6, and the roundings of the sum over 2 h
        assert abs(numeric - (gx.double() * d.double()).sum().item()) <= 1e-3 * (gx * d).abs().sum().item()


@pytest.mark.gpu
def test_stream_and_graph():
    """Captured forward and backward, replayed with the program's own work between, give what
    eager calls do."""
    from gfd.fused import group_norm
    w, b = affine(32, torch.float32)
    for shape, ptr in (((500, 32), None), ((3, 2000, 32), None),
                       ((5000, 32), torch.tensor([0, 10, 3000, 3000, 4990], device=DEV))):
        x, g = data(shape, torch.float32), data(shape, torch.float32, seed=9)

        def run():
            leaves = [t.detach().requires_grad_() for t in (x, w, b)]
            y = group_norm(leaves[0], 4, leaves[1], leaves[2], act="silu", ptr=ptr)
            return (y.detach(),) + torch.autograd.grad(y, leaves, g)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        for k in range(3):
            x.copy_(data(shape, torch.float32, seed=20 + k))
            want = run()
            graph.replay()
            torch.cuda.synchronize()
            for a, c in zip(out, want):
                assert torch.equal(a, c)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu"])
def test_a_group_of_one_element_has_no_gradient(act):
    """Its output is act(bias) wherever x is: w dz and its mean are one number."""
    from gfd.fused import group_norm
    w, b = affine(32, torch.float32)
    for x, ptr in ((data((60, 32), torch.float32), None), (data((7, 1, 3), torch.float32), None),
                   (data((60, 32), torch.float32), torch.arange(61, device=DEV))):
        C = x.shape[-1]
        xr, wr = x.requires_grad_(), w[:C].detach().requires_grad_()
        y = group_norm(xr, C, wr, b[:C], act=act, ptr=ptr)
        gx, gw = torch.autograd.grad(y, (xr, wr), data(x.shape, torch.float32, seed=5))
        assert not gx.any() and not gw.any()


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """The last rows of more than 2^31 elements give what they give alone: rows of their own, two
    long segments, and short ones behind a long one."""
    from gfd.fused import group_norm
    rows = 2 ** 31 // 64 + 100002
    x = torch.empty((rows, 64), dtype=torch.bfloat16, device=DEV).normal_()
    w, b = affine(64, torch.float32)

    def run(x, g, ptr=None):
        xr = x.detach().requires_grad_()
        y = group_norm(xr, 8, w, b, act="silu", ptr=ptr)
        return y.detach(), torch.autograd.grad(y, xr, g)[0]

    g = torch.empty_like(x).normal_()
    for whole, last in (((x, g), slice(-1000, None)), ((x.view(2, -1, 64), g.view(2, -1, 64)), slice(1, None))):
        for a, c in zip(run(*whole), run(*(t[last] for t in whole))):
            assert torch.equal(a[last], c)
    ptr = torch.tensor([0, rows - 5000, rows - 4990, rows - 2, rows], device=DEV)
    y, gx = run(x, g, ptr)
    tail = x[-5000:]
    ry, size, rx, _, _, back = reference(tail, 8, w, b, 1e-5, "silu", [10, 4988, 2], g[-5000:])
    assert ((y[-5000:].cpu().double() - ry).abs() <= OPS * size + 2.0 ** -8 * ry.abs()).all()
    scale = 1.2 * w.abs().max().item() * g[-5000:].abs().max().item() * (1 + size.max().item())
    assert ((gx[-5000:].cpu().double() - rx).abs() <= OPS * scale * 3 * back + 2.0 ** -8 * rx.abs()).all()


@pytest.mark.gpu
def test_same_result_twice():
    from gfd.fused import group_norm
    x, g = data((5000, 64), torch.bfloat16), data((5000, 64), torch.bfloat16, seed=4)
    ptr = torch.tensor([0, 1, 700, 701, 4000, 5000], device=DEV)
    outs = []
    for _ in range(2):
        leaves = [t.detach().requires_grad_() for t in (x, *affine(64, torch.float32))]
        y = group_norm(leaves[0], 8, leaves[1], leaves[2], act="gelu", ptr=ptr)
        outs.append((y,) + torch.autograd.grad(y, leaves, g))
    for a, c in zip(*outs):
        assert torch.equal(a, c)


@pytest.mark.gpu
def test_refused_on_the_device():
    from gfd.fused import group_norm
    x = torch.zeros((4, 8), device=DEV)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        group_norm(x.double(), 2)
    with pytest.raises(TypeError, match="weight and bias"):
        group_norm(x, 2, torch.ones(8, device=DEV).bfloat16())
    with pytest.raises(TypeError, match="weight and bias"):
        group_norm(x.bfloat16(), 2, torch.ones(8, device=DEV), torch.ones(8, device=DEV).bfloat16())
    with pytest.raises(RuntimeError, match="weight is on cpu"):
        group_norm(x, 2, torch.ones(8))
    with pytest.raises(ValueError, match="weight must be"):
        group_norm(x, 2, torch.ones(4, device=DEV))
    with pytest.raises(ValueError, match="multiple of 3 groups"):
        group_norm(x, 3)
    with pytest.raises(ValueError, match="act must be"):
        group_norm(x, 2, act="tanh")
    with pytest.raises(ValueError, match="x must be"):
        group_norm(x[0], 2)
    with pytest.raises(ValueError, match="ptr must be"):
        group_norm(x, 2, ptr=torch.tensor([0, 4], device=DEV, dtype=torch.int32))
    with pytest.raises(ValueError, match="with ptr"):
        group_norm(x[None], 2, ptr=torch.tensor([0, 4], device=DEV))
    with pytest.raises(ValueError, match="eps"):
        group_norm(x, 2, eps=-1.0)
    with pytest.raises(NotImplementedError, match="2048"):
        group_norm(torch.zeros((1, 2049), device=DEV), 1)
    xr = x.clone().requires_grad_()
    gx, = torch.autograd.grad(group_norm(xr, 2).sum(), xr, create_graph=True)
    with pytest.raises(RuntimeError):                         # no second derivative
        gx.sum().backward()


def test_refused_without_a_device():
    from gfd.fused import group_norm
    from gfd.nn import GroupNorm
    with pytest.raises(RuntimeError, match="HIP device"):
        group_norm(torch.zeros(4, 8), 2)
    with pytest.raises(ValueError, match="divisible"):
        GroupNorm(3, 8)
    with pytest.raises(ValueError, match="act"):
        GroupNorm(2, 8, act="swish")


def test_c_argument_errors():
    from gfd import _lib
    lib = _lib.load()
    size = lib.gfd_group_norm_workspace_size
    assert size(1, 100000, 0, 64, 8, 0) > 0 and size(200000, 1, 0, 64, 8, 0) == 0
    assert size(200000, 1, 0, 64, 8, 1) > 0 and size(4, 100, 1, 64, 8, 1) > 0 and size(4, 100, 1, 64, 8, 0) > 0
    assert size(1, 10, 0, 64, 7, 0) == 0

    def fwd(dtype=0, channels=8, groups=2, w_dtype=0, eps=1e-5, act=0, x=256, y=256, segments=1, length=4,
            stride=8):
        return lib.gfd_group_norm_fwd(x, dtype, segments, length, None, channels, groups, stride, 0, None,
                                      None, w_dtype, eps, act, y, None, None, 0, None)
    assert fwd(dtype=3) == 1 and fwd(groups=3) == 1 and fwd(eps=-1.0) == 1 and fwd(act=4) == 1
    assert fwd(x=None) == 1 and fwd(y=None) == 1 and fwd(x=258) == 1 and fwd(w_dtype=1) == 1
    assert fwd(channels=4096, groups=1) == 5 and fwd(segments=-1) == 1 and fwd(stride=-8) == 1
    assert fwd(length=0) == 0 and fwd(segments=0) == 0         # nothing to do
    assert fwd(length=100000) == 3                             # no workspace


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu"])
@pytest.mark.parametrize("shape", [(1, 64), (5, 64), (300, 32), (4100, 24), (17, 1, 24), (70, 15), (9, 40, 24),
                                   (2, 3000, 16)])
def test_an_eps_of_zero(shape, act):
    """Outputs and all gradients, at row counts that leave the last blocks' rows in part unused."""
    C = shape[-1]
    for dtype in (torch.float32, torch.bfloat16):
        check(data(shape, dtype), C // 8 if C % 8 == 0 else 3, *affine(C, torch.float32), act=act, eps=0.0)
        check(data(shape, dtype), C // 8 if C % 8 == 0 else 3, *affine(C, torch.float32), act=act, eps=1e-60)


@pytest.mark.gpu
@pytest.mark.parametrize("level", [2.0 ** 17, 2.0 ** 20, -2.0 ** 22])
@pytest.mark.parametrize("act", ["none", "relu"])
def test_levels_far_above_the_spread(level, act):
    """Up to where a step of fp32 is a third of the spread: rows, groups of three of a row, short
    and long dense segments, ragged ones of both kinds."""
    for shape, groups in (((300, 64), 8), ((64, 24), 8), ((5, 30, 24), 4), ((3, 4000, 24), 4)):
        check(data(shape, torch.float32, level=level), groups, *affine(shape[-1], torch.float32), act=act)
    lens = [3, 0, 40, 700, 1, 31]
    check(data((780, 24), torch.float32, level=level), 4, *affine(24, torch.float32), act=act, lens=lens,
          ptr=torch.tensor([0] + lens).cumsum(0).to(DEV))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(40, 24), (5, 30, 24), (3, 4000, 24)])
def test_a_constant_far_from_zero(shape):
    """Its variance is 0, not what squares of it would leave: the output is the bias, the gradient
    1 / sqrt(eps) times the centred w dy."""
    x = torch.full(shape, 1e6, device=DEV)
    y = check(x, 8, *affine(24, torch.float32))
    assert torch.equal(y.detach(), affine(24, torch.float32)[1].expand(shape))


def test_workspace_of_the_largest_shapes():
    """Sizes whose rows leave 31 or 63 bits are answered, and a call with more tiles than a launch
    counts is refused."""
    from gfd import _lib
    lib = _lib.load()
    for segments, length in ((2, 1 << 40), (65535, 1 << 40), (1 << 40, 1 << 40), (65536, 1 << 40)):
        for backward in (0, 1):
            assert lib.gfd_group_norm_workspace_size(segments, length, 0, 64, 8, backward) >= 0
    assert lib.gfd_group_norm_workspace_size(2, 1 << 40, 1, 64, 8, 1) > 0
    for ptr in (None, 256):
        assert lib.gfd_group_norm_fwd(256, 0, 2, 1 << 40, ptr, 64, 8, 64, 0, None, None, 0, 1e-5, 0, 256, None,
                                      None, 0, None) == 5


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_gelu_to_its_type(dtype):
    """Through a norm that changes nothing (groups of +-1, eps 0) z is the weight: the activation
    and its derivative over -9 .. 9.  fp32: within 4 roundings of 2^-24 of z and of 1.13, its
    largest slope.  fp16: half a step and a tenth, in the tail too."""
    from gfd.fused import group_norm
    C = 2048
    z = torch.linspace(-9, 9, C, device=DEV).to(dtype).float()
    sign = torch.where(torch.arange(C, device=DEV) % 2 == 0, 1.0, -1.0)
    x = sign.expand(3, C).to(dtype).requires_grad_()
    b = torch.zeros(C, device=DEV, requires_grad=True)
    y = group_norm(x, 1, (z * sign).requires_grad_(), b, 0.0, "gelu")
    db, = torch.autograd.grad(y, b, torch.ones_like(y) / 4)
    z = z.cpu().double()
    phi = 0.5 * torch.special.erfc(-z * 0.5 ** 0.5)
    want = z * phi
    slope = phi + z * torch.exp(-z * z / 2) / (2 * torch.pi) ** 0.5
    err = (y[0].detach().cpu().double() - want).abs()
    if dtype == torch.float32:
        assert (err <= 4 * U * z.abs().clamp(min=U)).all(), (err / U / z.abs()).max().item()
    else:
        tiny = torch.finfo(dtype).smallest_normal
        assert (err <= 1.1 * torch.finfo(dtype).eps / 2 * want.abs().clamp(min=tiny)).all()
    # the sum of three, halved twice: 3 roundings more
    assert ((db.cpu().double() * 4 / 3 - slope).abs() <= 8 * U).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_served(dtype):
    """Without gradients (the tiles' statistics go through the workspace): the formula's values,
    and those with gradients to the bit, of rows, short and long dense segments, and a ragged
    batch of both."""
    from gfd.fused import group_norm
    lens = [3, 0, 40, 2000, 1, 31, 700]
    ptr = torch.tensor([0] + lens).cumsum(0).to(DEV)
    w, b = affine(24, torch.float32)
    for shape, at in (((300, 24), None), ((9, 40, 24), None), ((2, 3000, 24), None), ((sum(lens) + 3, 24), ptr)):
        x = data(shape, dtype)
        with torch.no_grad():
            y = group_norm(x, 4, w, b, act="silu", ptr=at)
        ry, size = reference(x, 4, w, b, 1e-5, "silu", lens if at is not None else None)
        assert ((y.cpu().double() - ry).abs() <= OPS * size + half_step(dtype) * ry.abs()).all()
        assert torch.equal(y, group_norm(x, 4, w.detach().requires_grad_(), b, act="silu", ptr=at))


@pytest.mark.gpu
def test_gelu_of_ordinary_fp32_values():
    """Two roundings, of Phi and of the product: their deviations, 2^-24 / sqrt 3 each at most, are
    4.9e-8 of the values together, where an erf within 1.5e-7 of itself comes to 8.6e-8."""
    from gfd.fused import group_norm
    C = 2048
    z = (torch.randn(C, generator=torch.Generator().manual_seed(3)) * 1.2).to(DEV)
    sign = torch.where(torch.arange(C, device=DEV) % 2 == 0, 1.0, -1.0)
    y = group_norm(sign[None], 1, z * sign, None, 0.0, "gelu")[0].cpu().double()
    z = z.cpu().double()
    want = z * 0.5 * torch.special.erfc(-z * 0.5 ** 0.5)
    assert ((y - want).norm() / want.norm()).item() <= 6e-8
