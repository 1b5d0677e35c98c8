"""Log probabilities of given classes with entropy and top alternatives
(gfd.fused.class_log_probs): the HIP kernels against the formula in 64 bits,
forward and backward; and what it refuses.

Tolerances count roundings of U = 2^-24: a logit's exponential carries its
exponent's (a few for each unit of it), a lane adds classes / 64 of them at
most one after the other, and the logarithm, the subtractions and the final
division are under 64 in all."""
import pytest
import torch

DEV = "cuda"
U = 2.0 ** -24
INF = float("inf")


def reference(x, target, top, ignore=-1):
    x = x.detach().cpu().double()
    m = x.amax(1, keepdim=True)
    empty = (m == -INF)[:, 0]
    m = torch.where(m == -INF, torch.zeros_like(m), m)
    e = (x - m).exp()
    s = e.sum(1, keepdim=True)
    logp = torch.where(empty[:, None], torch.full_like(x, -INF), x - m - s.log())
    lost = x.isnan().any(1) | (x == INF).any(1)   # NaN throughout
    logp = torch.where(lost[:, None], torch.full_like(x, float("nan")), logp)
    p = torch.where(empty[:, None], torch.zeros_like(x), e / s)
    p = torch.where(lost[:, None], torch.full_like(x, float("nan")), p)
    h = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(1)
    h = torch.where(lost, torch.full_like(h, float("nan")), h)
    order = torch.sort(x + 0.0, dim=1, descending=True, stable=True).indices[:, :top]
    given = None
    if target is not None:
        t = target.cpu()
        given = logp.gather(1, t.clamp(0, x.shape[1] - 1)[:, None])[:, 0]
        given = torch.where((t < 0) | (t >= x.shape[1]), torch.full_like(given, float("nan")), given)
        given = torch.where(t == ignore, torch.zeros_like(given), given)
    return logp, p, h, given, order


def same(got, want, bound, what):
    got = got.detach().cpu().double()
    fine = want.isfinite()
    assert torch.equal(got[~fine].nan_to_num(7.0), want[~fine].nan_to_num(7.0)), what
    err = (got - want).abs()
    assert (err[fine] <= bound.expand_as(want)[fine]).all(), (what, err[fine].max().item())


def check(x, target, top, ignore=-1, seed=0, with_top_grad=True):
    from gfd.fused import class_log_probs
    xr = x.detach().requires_grad_()
    r = class_log_probs(xr, target, top, ignore)
    N, V = x.shape
    logp, p, h, given, order = reference(x, target, top, ignore)
    base = U * (64 + V / 64)
    size = torch.where(logp.isfinite(), logp.abs(), torch.zeros_like(logp))
    sound = ~x.detach().cpu().isnan().any(1)      # of a row with a NaN, some classes are listed
    assert torch.equal(r.top_classes.cpu()[sound], order[sound]), "classes"
    assert ((r.top_classes >= 0) & (r.top_classes < V)).all()
    want = logp.gather(1, order)
    same(r.top_log_probs, want, base + 4 * U * size.gather(1, order), "top")
    same(r.entropy, h, base * (10 + h), "entropy")
    if target is not None:
        same(r.log_prob, given, base + 4 * U * given.nan_to_num(0, 0, 0).abs(), "given")
    g = torch.Generator().manual_seed(seed)
    gl, ge, gt = (torch.randn(s, generator=g) for s in ((N,), (N,), (N, top)))
    outs, grads = [r.entropy], [ge]
    total = torch.zeros(N, dtype=torch.float64)
    extra = torch.zeros(N, V, dtype=torch.float64)
    if target is not None:
        t = target.cpu()
        known = t != ignore
        outs.append(r.log_prob)
        grads.append(gl)
        total += torch.where(known, gl.double(), torch.zeros(N, dtype=torch.float64))
        extra.scatter_add_(1, t.clamp(0, V - 1)[:, None], (gl.double() * known)[:, None])
        total = torch.where(known & ((t < 0) | (t >= V)), torch.full_like(total, float("nan")), total)
    if top and with_top_grad:
        outs.append(r.top_log_probs)
        grads.append(gt)
        total += gt.double().sum(1)
        extra.scatter_add_(1, order, gt.double())
    inner = torch.where(p > 0, logp, torch.zeros_like(p)) + h[:, None]
    ref = -p * (total[:, None] + ge.double()[:, None] * inner) + extra
    ref[(x.detach().cpu() == -INF).all(1)] = 0
    got, = torch.autograd.grad(outs, xr, [t.to(DEV) for t in grads])
    assert got.dtype == x.dtype
    part = p * (total.nan_to_num()[:, None].abs() + gt.abs().double().sum(1)[:, None] +
                ge.double()[:, None].abs() * (inner.abs() + 10 + h[:, None]))
    step = U if x.dtype == torch.float32 else torch.finfo(x.dtype).eps / 2
    bound = (base + 4 * U * size) * part + 8 * U * (extra.abs() + gt.abs().double().sum(1)[:, None])
    same(got, ref, bound + step * ref.abs().nan_to_num() + torch.finfo(x.dtype).tiny, "gradient")
    return r


def logits(N, V, dtype, seed=0, std=2.0):
    return (torch.randn((N, V), generator=torch.Generator().manual_seed(seed)) * std).to(dtype).to(DEV)


def targets(N, V, seed=1):
    t = torch.randint(V, (N,), generator=torch.Generator().manual_seed(seed))
    t[::5] = -1
    return t.to(DEV)


SIZES = [1, 2, 3, 4, 5, 15, 16, 17, 63, 64, 65, 127, 128, 129, 511, 512, 513, 1000, 4095, 4096, 4097, 5001, 8191, 20000]


@pytest.mark.gpu
@pytest.mark.parametrize("V", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_classes(V, dtype):
    check(logits(11, V, dtype), targets(11, V), min(V, 5))


@pytest.mark.gpu
@pytest.mark.parametrize("N,V", [(1, 1), (1, 100000), (2, 70001), (5000, 2), (3001, 7), (1500, 130), (1100, 4500),
                                 (1100, 3000), (4100, 4200), (520, 6000)])
def test_rows(N, V):
    check(logits(N, V, torch.float32), targets(N, V), min(V, 3))


@pytest.mark.gpu
@pytest.mark.parametrize("top", [0, 1, 2, 31, 32, 33, 63, 64])
@pytest.mark.parametrize("V", [64, 100, 700, 9000, 300000])
def test_top(top, V):
    check(logits(6, V, torch.bfloat16), targets(6, V), top)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [10, 128, 300, 6000, 50000])
def test_ties_and_orders(V):
    """Equal logits, -0 and +0, rising rows (every logit enters the list) and falling ones."""
    k = min(V, 40)
    few = torch.randint(3, (4, V), generator=torch.Generator().manual_seed(4)).float().to(DEV)
    check(few, targets(4, V), k)
    check(torch.zeros((3, V), device=DEV), targets(3, V), k)
    check(torch.where(torch.arange(V, device=DEV) % 2 == 0, 0.0, -0.0).expand(3, V).contiguous(), targets(3, V), k)
    ramp = torch.linspace(-9, 9, V, device=DEV).expand(3, V).contiguous()
    check(ramp, targets(3, V), k)
    check(ramp.flip(1).contiguous(), targets(3, V), k)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [7, 128, 700, 6000, 50000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_masked(V, dtype):
    x = logits(8, V, dtype)
    gone = torch.rand((8, V), generator=torch.Generator().manual_seed(5)).to(DEV) < 0.7
    x.masked_fill_(gone, -INF)
    x[1] = -INF                                   # no class left
    x[2] = -INF
    x[2, V - 1] = 1.0                             # one left: the last
    x[3] = torch.finfo(dtype).min                 # the type's lowest value: uniform
    x[4, : V // 2] = torch.finfo(dtype).min
    r = check(x, targets(8, V), min(V, 9))
    assert r.entropy[1] == 0 and r.entropy[2] == 0


@pytest.mark.gpu
@pytest.mark.parametrize("V", [7, 128, 700, 6000, 50000])
def test_nan_and_infinity_stay_in_their_row(V):
    from gfd.fused import class_log_probs
    x = logits(6, V, torch.float32)
    x[1, V // 2] = float("nan")
    x[3, V - 1] = INF
    x[4] = float("nan")
    x[5, 0], x[5, 1:] = float("nan"), -INF
    t = torch.zeros(6, dtype=torch.int64, device=DEV)
    xr = x.requires_grad_()
    r = class_log_probs(xr, t, min(V, 4))
    g, = torch.autograd.grad(r.log_prob.sum() + r.entropy.sum(), xr)
    bad = torch.tensor([False, True, False, True, True, True])
    assert torch.equal(r.entropy.isnan().cpu(), bad) and torch.equal(r.log_prob.isnan().cpu(), bad)
    assert torch.equal(r.top_log_probs.isnan().all(1).cpu(), bad)
    assert torch.equal(g.isnan().all(1).cpu(), bad) and torch.equal(g.isnan().any(1).cpu(), bad)
    assert ((r.top_classes >= 0) & (r.top_classes < V)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("V", [6, 600, 9000])
def test_far_and_confident_logits(V):
    x = logits(5, V, torch.float32)
    x[0] += 3e4                                   # a level far from 0
    x[1, 2] = 80.0                                # the rest adds next to nothing
    x[2] *= 40
    x[3] = torch.linspace(-3e38, 3e38, V)         # its step overflows: infinities and NaN
    check(x, torch.full((5,), 2, device=DEV), 3)
    x[3] = torch.linspace(-1.6e38, 1.6e38, V)
    check(x, torch.full((5,), 2, device=DEV), 3)


@pytest.mark.gpu
def test_targets():
    from gfd.fused import class_log_probs
    for V in (5, 700, 9000):
        x = logits(6, V, torch.float32)
        t = torch.tensor([-1, -2, 0, V - 1, V, 2 ** 62], device=DEV)
        check(x, t, 2)
        check(x, t, 2, ignore=0)
        check(x, t, 0, ignore=-100)
        check(x, None, 2)
    assert class_log_probs(x).log_prob is None


@pytest.mark.gpu
@pytest.mark.parametrize("V", [9, 600, 5000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides(V, dtype):
    base = logits(20, V + 24, dtype)
    for off in (0, 8, 3):
        check(base[:, off:off + V], targets(20, V), 3)
        check(base[::3, off:off + V], targets(7, V), 3)
    check(base.t().contiguous().t()[:, :V], targets(20, V), 3)
    check(base[:1, :V].expand(20, V), targets(20, V), 3)


@pytest.mark.gpu
def test_shapes():
    from gfd.fused import class_log_probs
    x = logits(6, 10, torch.float32)
    r = class_log_probs(x.view(2, 3, 10), targets(6, 10).view(2, 3), 4)
    flat = class_log_probs(x, targets(6, 10), 4)
    assert r.log_prob.shape == r.entropy.shape == (2, 3) and r.top_classes.shape == (2, 3, 4)
    assert torch.equal(r.log_prob.view(-1), flat.log_prob)
    one = class_log_probs(x[0], torch.tensor(3, device=DEV), 1)
    assert one.log_prob.shape == () and one.top_classes.shape == (1,)
    none = class_log_probs(x[:0], targets(6, 10)[:0], 2)
    assert none.log_prob.shape == (0,) and none.top_log_probs.shape == (0, 2)
    xr = x[:0].detach().requires_grad_()
    assert torch.autograd.grad(class_log_probs(xr).entropy.sum(), xr)[0].shape == (0, 10)


@pytest.mark.gpu
def test_gradient_against_differences():
    from gfd.fused import class_log_probs
    x, t = logits(4, 30, torch.float32), targets(4, 30)

    def f(v):
        r = class_log_probs(v, t, 3)
        return r.log_prob.sum() + 2 * r.entropy.sum() + 0.5 * r.top_log_probs.sum()
    xr = x.clone().requires_grad_()
    g, = torch.autograd.grad(f(xr), xr)
    d = logits(4, 30, torch.float32, seed=8, std=1.0)
    h = 2.0 ** -9
    numeric = (f(x + h * d).double() - f(x - h * d).double()).item() / (2 * h)
    assert abs(numeric - (g * d).sum().item()) <= 2e-3 * (g * d).abs().sum().item()


@pytest.mark.gpu
def test_loss_alone_is_cross_entropy():
    """-log_prob summed over the known labels is the cross entropy with ignore_index."""
    from gfd.fused import class_log_probs
    x, t = logits(200, 12, torch.float32).requires_grad_(), targets(200, 12)
    loss = -class_log_probs(x, t).log_prob.sum()
    g, = torch.autograd.grad(loss, x)
    xd = x.detach().cpu().double().requires_grad_()
    ref = torch.nn.functional.cross_entropy(xd, t.cpu(), ignore_index=-1, reduction="sum")
    gd, = torch.autograd.grad(ref, xd)
    assert abs(loss.item() - ref.item()) <= 200 * 80 * U * 4
    assert (g.cpu().double() - gd).abs().max() <= 100 * U


@pytest.mark.gpu
def test_stream_and_graph():
    from gfd.fused import class_log_probs
    for N, V in ((300, 6), (40, 900), (2, 60000)):
        x, t = logits(N, V, torch.float32), targets(N, V)
        gl, ge, gt = (torch.randn(s, device=DEV) for s in ((N,), (N,), (N, 4)))

        def run():
            xr = x.detach().requires_grad_()
            r = class_log_probs(xr, t, 4)
            g, = torch.autograd.grad((r.log_prob, r.entropy, r.top_log_probs), xr, (gl, ge, gt))
            return r.log_prob.detach(), r.entropy.detach(), r.top_log_probs.detach(), r.top_classes, g

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        for k in range(3):
            x.copy_(logits(N, V, torch.float32, seed=30 + k))
            want = run()
            graph.replay()
            torch.cuda.synchronize()
            for a, c in zip(out, want):
                assert torch.equal(a, c)


@pytest.mark.gpu
def test_refused_on_the_device():
    from gfd.fused import class_log_probs
    x = torch.zeros((4, 8), device=DEV)
    t = torch.zeros(4, dtype=torch.int64, device=DEV)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        class_log_probs(x.double(), t)
    with pytest.raises(TypeError, match="int64"):
        class_log_probs(x, t.int())
    with pytest.raises(ValueError, match="target must be"):
        class_log_probs(x, t[:3])
    with pytest.raises(RuntimeError, match="target is on cpu"):
        class_log_probs(x, t.cpu())
    for top in (-1, 9):
        with pytest.raises(ValueError, match="top must be"):
            class_log_probs(x, t, top)
    with pytest.raises(ValueError, match="top must be"):
        class_log_probs(torch.zeros((1, 100), device=DEV), None, 65)
    with pytest.raises(ValueError, match="classes"):
        class_log_probs(torch.zeros((4, 0), device=DEV))


def test_refused_without_a_device():
    from gfd.fused import class_log_probs
    from gfd.models import GAT
    with pytest.raises(RuntimeError, match="HIP device"):
        class_log_probs(torch.zeros(4, 8))
    with pytest.raises(ValueError, match="out_channels"):
        GAT(5, 64, 1).log_probs(torch.zeros(2, 5), None)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """The last rows of more than 2^31 logits give what they give alone."""
    from gfd.fused import class_log_probs
    V = 203769
    rows = 2 ** 31 // V + 700
    x = torch.empty((rows, V), dtype=torch.bfloat16, device=DEV).normal_()
    t = torch.randint(V, (rows,), generator=torch.Generator().manual_seed(4)).to(DEV)

    def run(x, t):
        xr = x.detach().requires_grad_()
        r = class_log_probs(xr, t, 4)
        gx, = torch.autograd.grad((r.log_prob.sum(), r.entropy.sum(), r.top_log_probs[:, 1].sum()), xr)
        return tuple(o.detach() for o in r) + (gx,)

    for a, c in zip(run(x, t), run(x[-600:], t[-600:])):
        assert torch.equal(a[-600:], c)


def test_c_argument_errors():
    from gfd import _lib
    lib = _lib.load()
    size = lib.gfd_class_logp_workspace_size
    assert size(1, 200000, 10) > size(1, 200000, 0) > 0
    assert size(100000, 200, 10) == 0 and size(1, 10, 11) == 0

    def fwd(x=256, dtype=0, rows=2, classes=8, target=256, top=0, logp=256, ent=256, tl=256, tc=256, stats=256):
        return lib.gfd_class_logp_fwd(x, dtype, rows, classes, classes, target, -1, top, logp, ent, tl, tc,
                                      stats, None, 0, None)
    assert fwd(rows=0) == 0
    assert fwd(dtype=3) == 1 and fwd(classes=0) == 1 and fwd(top=9) == 1 and fwd(top=-1) == 1
    assert fwd(classes=100, top=65) == 1 and fwd(classes=2 ** 31) == 1
    assert fwd(x=None) == 1 and fwd(x=258) == 1 and fwd(target=None) == 1 and fwd(ent=None) == 1
    assert fwd(top=2, tc=None) == 1 and fwd(stats=None) == 1
    assert fwd(classes=200000) == 3                            # no workspace


@pytest.mark.gpu
@pytest.mark.parametrize("V", [20, 130, 700, 5000, 70001])
@pytest.mark.parametrize("N", [3, 1500])
def test_statistics_are_the_maximum_and_the_log_sum(N, V):
    """As include/gfd.h states them, also of a row whose largest logit follows some that lie less
    than its sums' slack below it, and of a confident one; log probabilities are not above 0,
    entropies not below it."""
    from gfd import fused
    x = torch.full((N, V), -50.0)
    x[:, ::2] = 0.0
    x[:, V // 2 + 1::max(V // 5, 1)] = 7.5
    x[1] = -90.0
    x[1, V - 1] = 12.25
    x[2] = torch.randn(V, generator=torch.Generator().manual_seed(2)) * 3
    t = x.argmax(1)
    m = x.double().amax(1)
    ls = (x.double() - m[:, None]).exp().sum(1).log()
    for top in (0, 3):
        logp, entropy, top_logp, _, stats = fused._class_log_probs_fwd(x.to(DEV), t.to(DEV), top, -1, True)[:5]
        assert torch.equal(stats[:, 0].cpu().double(), m)
        # a sum's roundings, and those of exponents up to 16 in it
        assert ((stats[:, 1].cpu().double() - ls).abs() <= U * (64 + V / 64)).all()
        assert (logp <= 0).all() and (entropy >= 0).all() and (top_logp <= 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("N", [1, 2, 33])
@pytest.mark.parametrize("V", [20, 700, 70001, 300000])
def test_served(N, V):
    """Without gradients (no statistics kept, the split rows' beside the partial lists): the
    reference's values, and those with gradients to the bit."""
    from gfd.fused import class_log_probs
    x = logits(N, V, torch.bfloat16, seed=N)
    for target, top in ((targets(N, V), 0), (targets(N, V), 7), (None, 0), (None, 64 if V > 64 else 3)):
        with torch.no_grad():
            r = class_log_probs(x, target, top)
        logp, _, h, given, order = reference(x, target, top)
        base = U * (64 + V / 64)
        assert torch.equal(r.top_classes.cpu(), order)
        want = logp.gather(1, order)
        same(r.top_log_probs, want, base + 4 * U * want.abs(), "top")
        same(r.entropy, h, base * (10 + h), "entropy")
        if target is not None:
            same(r.log_prob, given, base + 4 * U * given.abs(), "given")
        for a, b in zip(r, class_log_probs(x.detach().requires_grad_(), target, top)):
            assert a is b is None or torch.equal(a, b) and not a.requires_grad
