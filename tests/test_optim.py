"""Adam and AdamW over many tensors (gfd.optim): the HIP kernel against the
formulas in 64 bits, states in 32 and in 8 bits; the optimizer as torch's; and
what it refuses.

Tolerances count roundings of U = 2^-24.  32-bit states: a moment is two
products and a sum (4 U of its terms); the update takes the root, the division,
the two corrections and the rate (16 U of itself) and is subtracted from the
parameter, which is rounded to its type (half a step).  8-bit states are
exact: a code is a function of the moment in fp32, and that is fp64 rounded
once."""
import copy
import math

import pytest
import torch

DEV = "cuda"
U = 2.0 ** -24
BLOCK = 256


def make(sizes, dtype, seed=0, offset=0):
    """Parameters with gradients; offset: their first element's place in an allocation."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for s in sizes:
        n = math.prod(s) if isinstance(s, tuple) else s
        p = torch.zeros(n + offset, dtype=dtype, device=DEV)[offset:]
        p.copy_(torch.randn(n, generator=g) * 0.1)
        p = p.view(s) if isinstance(s, tuple) else p
        p.requires_grad_()
        grad = torch.zeros(n + offset, dtype=dtype, device=DEV)[offset:]
        p.grad = grad.copy_(torch.randn(n, generator=g) * 0.02).view(p.shape)
        out.append(p)
    return out


def moments(opt, p):
    """(m, v) of a parameter in fp64, as its states stand."""
    s = opt.state[p]
    m, v = s["exp_avg"].detach().cpu(), s["exp_avg_sq"].detach().cpu()
    if "exp_avg_scale" not in s:
        return m.double(), v.double()
    n = p.numel()
    scale = [s[k].cpu().double().repeat_interleave(BLOCK)[:n].view(p.shape)
             for k in ("exp_avg_scale", "exp_avg_sq_scale")]
    return m.double() * scale[0], (v.double() * scale[1]) ** 2


def formula(p, g, m, v, t, lr, b1, b2, eps, wd, decoupled):
    p, g = p.double(), g.double()
    if decoupled:
        p = p * (1 - lr * wd)
    else:
        g = g + wd * p
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    change = lr / (1 - b1 ** t) * m / (v.sqrt() / math.sqrt(1 - b2 ** t) + eps)
    return p - change, m, v, change


def mix(h):
    for shift, mul in ((16, 0x7FEB352D), (15, 0x846CA68B)):
        h = (h ^ (h >> shift)) * mul & 0xFFFFFFFF
    return h ^ (h >> 16)


def codes(x, noise, floor):
    """(e4m3 values, scales) of fp32 values by the rule include/gfd.h states."""
    n = x.numel()
    pad = torch.zeros(-(-n // BLOCK) * BLOCK, dtype=torch.float64)
    pad[:n] = x.double().reshape(-1)
    blocks = pad.view(-1, BLOCK)
    top = blocks.abs().amax(1)
    e = torch.where(top > 0, torch.floor(torch.log2(top.clamp(min=1e-300))) - 7, torch.full_like(top, -100))
    scale = torch.exp2(e.clamp(min=-100))
    a = (blocks / scale[:, None]).view(-1)[:n].abs()
    step = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3)
    c = torch.floor(a / step + noise.double() / 65536) * step
    if floor:
        c = torch.where((c == 0) & (a > 0), torch.full_like(c, 2.0 ** -9), c)
    return (c * torch.sign(x.double().reshape(-1))).view(x.shape), scale


def random_bits(first, n, t, seed):
    key = mix((mix(t) + seed) & 0xFFFFFFFF)
    place = (torch.arange(first, first + n, dtype=torch.int64) * 0x9E3779B1 + key) & 0xFFFFFFFF
    u = place.clone()
    for shift, mul in ((16, 0x7FEB352D), (15, 0x846CA68B)):
        u = u ^ (u >> shift)
        lo = ((u & 0xFFFF) * mul + ((((u >> 16) * mul) & 0xFFFF) << 16)) & 0xFFFFFFFF
        u = lo
    u = u ^ (u >> 16)
    return u & 0xFFFF, u >> 16


SIZES = [1, 7, 255, 256, 257, 2047, 2048, 2049, (33, 7), (3, 5, 11), 70000]


def check_step(opt, params, cls, bits, lr=1e-2, betas=(0.9, 0.99), eps=1e-8, wd=0.1, seed=5, t=1):
    before = [(p.detach().cpu().clone(), p.grad.cpu().clone(), *moments(opt, p)) for p in params]
    opt.step()
    first = 0
    for p, (p0, g, m0, v0) in zip(params, before):
        p1, m1, v1, change = formula(p0, g, m0, v0, t, lr, *betas, eps, wd, cls == "AdamW")
        half = torch.finfo(p.dtype).eps / 2 if p.dtype != torch.float32 else U
        terms = betas[0] * m0.abs() + (1 - betas[0]) * (g.double().abs() + wd * p0.double().abs())
        # the moment is off by 4 U of its terms, which may cancel in it, and that goes through
        # the update's factor as it does itself
        factor = lr / (1 - betas[0] ** t) / (v1.sqrt() / math.sqrt(1 - betas[1] ** t) + eps)
        bound = (16 * U * (change.abs() + p1.abs()) + 4 * U * factor * terms + half * p1.abs() +
                 torch.finfo(p.dtype).tiny)
        assert ((p.detach().cpu().double() - p1).abs() <= bound).all()
        assert opt.state[p]["step"].item() == t
        if bits == 32:
            m, v = moments(opt, p)
            assert ((m - m1).abs() <= 4 * U * terms + 1e-45).all()
            # g^2: the gradient with its decay is rounded before it is squared
            big = betas[1] * v0 + (1 - betas[1]) * (g.double().abs() + wd * p0.double().abs()) ** 2
            assert ((v - v1).abs() <= 8 * U * big + 1e-45).all()
        else:
            u, w = random_bits(first, p.numel(), t, seed)
            root = v1.float().sqrt()
            for key, x, noise in (("exp_avg", m1.float(), u), ("exp_avg_sq", root, w)):
                want, scale = codes(x, noise, key == "exp_avg_sq")
                assert torch.equal(opt.state[p][key + "_scale"].cpu().double(), scale), key
                assert torch.equal(opt.state[p][key].cpu().double(), want), key
        first += -(-p.numel() // BLOCK) * BLOCK


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("cls", ["Adam", "AdamW"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("offset", [0, 1])
def test_steps(dtype, cls, bits, offset):
    from gfd import optim
    params = make(SIZES, dtype, offset=offset)
    opt = getattr(optim, cls)(params, lr=1e-2, betas=(0.9, 0.99), weight_decay=0.1, state_bits=bits, seed=5)
    opt.flat_state(0)
    for t in range(1, 4):
        check_step(opt, params, cls, bits, t=t)
        for k, p in enumerate(params):
            p.grad.mul_(-0.7).add_(0.003 * k)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors(bits):
    """More than one launch holds, empty ones among them."""
    from gfd.optim import AdamW
    params = make([1 + (k * 37) % 900 for k in range(230)], torch.float32)
    empty = torch.empty((0, 4), device=DEV, requires_grad=True)
    empty.grad = torch.empty((0, 4), device=DEV)
    opt = AdamW(params[:100] + [empty] + params[100:], lr=1e-2, betas=(0.9, 0.99), weight_decay=0.1,
                state_bits=bits, seed=5)
    opt.flat_state(0)
    for t in (1, 2):
        check_step(opt, params, "AdamW", bits, t=t)
    assert opt.state[empty]["step"].item() == 2


@pytest.mark.gpu
def test_large_tensor_takes_several_rounds_of_blocks():
    from gfd.optim import Adam
    params = make([2048 * 2048 * 2 + 77, 3], torch.bfloat16)
    opt = Adam(params, lr=1e-2, betas=(0.9, 0.99), weight_decay=0.1, state_bits=32)
    opt.flat_state(0)
    check_step(opt, params, "Adam", 32)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """The last elements of a parameter of more than 2^32, and one behind it, are updated as they
    are alone (a first step's update does not depend on how its states are rounded)."""
    from gfd.optim import Adam
    n = 2 ** 32 + 5003
    p = torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    p.grad = torch.zeros_like(p)
    q, r = make([5003, 700], torch.bfloat16)
    p[-5003:] = q.detach()
    p.grad[-5003:] = q.grad
    s = r.detach().clone()
    s.grad = r.grad.clone()
    big = Adam([p.requires_grad_(), s.requires_grad_()], lr=0.05, state_bits=8)
    alone = Adam([q, r], lr=0.05, state_bits=8)
    big.step()
    alone.step()
    assert torch.equal(p[-5003:], q) and torch.equal(s, r) and not p[:-5003].any()
    m, v = (big.state[p][k][-5003:].float() for k in ("exp_avg", "exp_avg_sq"))
    assert m.ne(0).any() and v.ne(0).sum() == q.grad.ne(0).sum()
    assert not big.state[p]["exp_avg"][:1000].float().any()


@pytest.mark.gpu
def test_missing_gradients_are_skipped():
    from gfd.optim import Adam
    params = make([300, 40, 500], torch.float32)
    opt = Adam(params, lr=0.1)
    kept, params[1].grad = params[1].grad, None
    old = params[1].detach().clone()
    opt.step()
    opt.step()
    assert torch.equal(params[1], old)
    params[1].grad = kept
    opt.step()
    assert [opt.state[p]["step"].item() for p in params] == [3, 1, 3]
    ref = torch.nn.Parameter(old.cpu().double())
    ref.grad = kept.cpu().double()
    r = torch.optim.Adam([ref], lr=0.1)
    r.step()
    assert (params[1].detach().cpu().double() - ref.detach()).abs().max() <= 32 * U


@pytest.mark.gpu
@pytest.mark.parametrize("cls", ["Adam", "AdamW"])
def test_follows_torch(cls):
    """20 steps of two groups on a quadratic, against torch's in 64 bits: a step's error is
    16 U of an update (at most about lr) and U of the parameter, and the gradient carries it on."""
    from gfd import optim
    start = torch.randn(2000, generator=torch.Generator().manual_seed(3))
    a, b = (torch.nn.Parameter(start.to(DEV)) for _ in range(2))
    c, d = (torch.nn.Parameter(start.double()) for _ in range(2))
    args = dict(lr=1e-2, betas=(0.8, 0.95), weight_decay=0.02, eps=1e-6)
    ours = getattr(optim, cls)([{"params": [a]}, {"params": [b], "lr": 3e-2, "weight_decay": 0.0}], **args)
    ref = getattr(torch.optim, cls)([{"params": [c]}, {"params": [d], "lr": 3e-2, "weight_decay": 0.0}], **args)
    sched = [torch.optim.lr_scheduler.StepLR(o, 7, 0.5) for o in (ours, ref)]
    for _ in range(20):
        def loss():
            ours.zero_grad()
            v = (a ** 2).sum() + (b ** 4).sum()
            v.backward()
            return v
        ours.step(loss)
        ref.zero_grad()
        ((c ** 2).sum() + (d ** 4).sum()).backward()
        ref.step()
        for s in sched:
            s.step()
    for x, y in ((a, c), (b, d)):
        assert (x.detach().cpu().double() - y.detach()).abs().max() <= 20 * 64 * U * 4


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_layouts(bits):
    """A transposed parameter, and a gradient in another order than its parameter's."""
    from gfd.optim import AdamW
    base, = make([(40, 24)], torch.float32)
    out = []
    for how in range(3):
        p = base.detach().clone().t() if how == 1 else base.detach().t().contiguous()
        p = p.requires_grad_()
        g = base.grad.t() if how == 2 else torch.empty_like(p).copy_(base.grad.t())
        p.grad = g
        opt = AdamW([p], lr=0.1, state_bits=bits)
        opt.step()
        opt.step()
        out.append((p.detach(), opt.state[p]["exp_avg"].float()))
    assert torch.equal(out[0][0], out[2][0])
    if bits == 32:
        assert torch.equal(out[0][0], out[1][0]) and torch.equal(out[0][1], out[1][1])


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_graph_replays_are_steps(bits):
    from gfd.optim import AdamW
    lr = torch.tensor(1e-2, device=DEV)
    a, b = make([3000, 17], torch.float32), make([3000, 17], torch.float32)
    ours, eager = (AdamW(p, lr=lr, state_bits=bits, seed=9) for p in (a, b))
    with pytest.raises(RuntimeError, match="before capturing"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            ours.step()
    torch.cuda.synchronize()
    ours.step()
    eager.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ours.step()
    for k in range(4):
        lr.mul_(0.7)
        for p, q in zip(a, b):
            q.grad.copy_(p.grad.add_(0.01 * k))
        graph.replay()
        eager.step()
        torch.cuda.synchronize()
        for p, q in zip(a, b):
            assert torch.equal(p, q)
        for key, t in ours.flat_state(0).items():
            assert torch.equal(t.view(torch.uint8) if t.dtype.itemsize == 1 else t,
                               eager.flat_state(0)[key].view(torch.uint8) if t.dtype.itemsize == 1
                               else eager.flat_state(0)[key]), key
    assert ours.flat_state(0)["step"].tolist() == [5, 5]


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict_and_copies(bits, tmp_path):
    from gfd.optim import AdamW
    a = make(SIZES, torch.bfloat16)
    ours = AdamW(a, lr=1e-2, state_bits=bits, seed=3)
    ours.step()
    torch.save(ours.state_dict(), tmp_path / "opt.pt")
    others = []
    for how in ("load", "copy"):
        b = [p.detach().clone().requires_grad_() for p in a]
        if how == "load":
            other = AdamW(b, lr=5.0)
            other.load_state_dict(torch.load(tmp_path / "opt.pt", weights_only=True))
        else:
            other, b = copy.deepcopy((ours, a))
        for p, q in zip(a, b):
            q.grad = p.grad.clone()
        others.append((other, b))
    ours.step()
    for other, b in others:
        other.step()
        for p, q in zip(a, b):
            assert torch.equal(p, q)
            for k, t in ours.state[p].items():
                o = other.state[q][k]
                assert t.dtype == o.dtype and torch.equal(t.float(), o.float()), k


@pytest.mark.gpu
def test_loads_torch_states():
    from gfd.optim import Adam
    p, = make([(30, 9)], torch.float32)
    q = p.detach().cpu().double().requires_grad_()
    q.grad = p.grad.cpu().double()
    ref = torch.optim.Adam([q], lr=0.05, weight_decay=0.01)
    ref.step()
    p.data.copy_(q.detach())
    ours = Adam([p], lr=9.0)
    ours.load_state_dict(ref.state_dict())
    ref.step()
    ours.step()
    assert ours.state[p]["step"].item() == 2
    # the states and the parameter were rounded to fp32 once more: 4 U of an update of lr
    assert (p.detach().cpu().double() - q.detach()).abs().max() <= U * 4 + 32 * U * 0.05
    bad = copy.deepcopy(ref.state_dict())
    bad["param_groups"][0]["amsgrad"] = True
    with pytest.raises(NotImplementedError, match="amsgrad"):
        ours.load_state_dict(bad)
    eight = Adam([p], state_bits=8)
    eight.step()
    with pytest.raises(ValueError, match="number of parameter groups|different number"):
        Adam([{"params": [p]}, {"params": make([3], torch.float32)}]).load_state_dict(eight.state_dict())


def test_other_kind_of_decay_is_not_loaded():
    """A state dict of AdamW into Adam, or the other way, would train on with another rule."""
    from gfd.optim import Adam, AdamW
    p = torch.zeros(4, requires_grad=True)
    for ours, theirs in ((Adam([p], weight_decay=0.1), AdamW([p], weight_decay=0.1)),
                         (AdamW([p]), Adam([p])), (Adam([p]), torch.optim.AdamW([p]))):
        with pytest.raises(ValueError, match="of the other kind"):
            ours.load_state_dict(theirs.state_dict())
        assert ours.param_groups[0]["lr"] == 1e-3
    AdamW([p]).load_state_dict(torch.optim.AdamW([p]).state_dict())


@pytest.mark.gpu
def test_a_refused_state_dict_changes_nothing():
    from gfd.optim import Adam
    p, q = make([300, (7, 5)], torch.float32)
    opt, same = Adam([p, q], lr=0.1), Adam([r.detach().clone().requires_grad_() for r in (p, q)], lr=0.1)
    for r, s in zip(same.param_groups[0]["params"], (p, q)):
        r.grad = s.grad.clone()
    opt.step()
    same.step()
    bad = copy.deepcopy(opt.state_dict())
    bad["state"][1]["exp_avg"] = torch.zeros(3)
    bad["param_groups"][0]["lr"] = 7.0
    with pytest.raises(ValueError, match="exp_avg"):
        opt.load_state_dict(bad)
    opt.step()
    same.step()
    for r, s in zip(same.param_groups[0]["params"], (p, q)):
        assert torch.equal(r, s) and torch.equal(same.state[r]["exp_avg"], opt.state[s]["exp_avg"])


@pytest.mark.gpu
def test_eight_bits_round_without_bias():
    """65536 elements with one moment between two codes: their mean is the moment's, within six
    of the mean's deviations (half a code step over the root of their number)."""
    from gfd.optim import Adam
    n = 65536
    p = torch.zeros(n, device=DEV, requires_grad=True)
    p.grad = torch.full((n,), 0.1234567, device=DEV)
    opt = Adam([p], betas=(0.0, 0.0), state_bits=8)
    opt.step()
    m, v = moments(opt, p)
    g = p.grad[0].double().item()
    step = 2.0 ** -3 * g
    assert len(m.unique()) == 2 and (m - g).abs().max() <= step
    assert abs(m.mean().item() - g) <= 6 * step / 2 / math.sqrt(n)
    assert abs(v.sqrt().mean().item() - g) <= 6 * step / 2 / math.sqrt(n)


@pytest.mark.gpu
def test_eight_bits_special_values():
    from gfd.optim import Adam
    p = torch.zeros(1024, device=DEV, requires_grad=True)
    g = torch.full((1024,), 1e-3, device=DEV)
    g[:256] = 0.0                       # a block of zeros
    g[256] = 1e4                        # one that dwarfs the rest of its block
    g[512], g[513] = float("nan"), float("inf")
    p.grad = g
    opt = Adam([p], lr=0.1, state_bits=8)
    opt.step()
    s = opt.state[p]
    m, r = s["exp_avg"].float(), s["exp_avg_sq"].float()
    assert not m[:256].any() and not r[:256].any() and torch.equal(p[:256], torch.zeros_like(p[:256]))
    assert (r[256:512] > 0).all()       # a root that is not 0 never becomes 0
    assert m[512:514].isnan().all() and r[512:514].isnan().all()
    assert m[514:].isfinite().all() and r[514:].isfinite().all() and p[514:].isfinite().all()
    opt.step()
    assert p[514:].isfinite().all() and p[:512].isfinite().all()


@pytest.mark.gpu
def test_tiny_and_huge_gradients():
    from gfd.optim import Adam
    for bits in (32, 8):
        p = torch.ones(512, device=DEV, requires_grad=True)
        p.grad = torch.cat([torch.full((256,), 1e-25), torch.full((256,), 1e15)]).to(DEV)
        opt = Adam([p], lr=0.1, state_bits=bits)
        for _ in range(3):
            opt.step()
        assert p.isfinite().all() and (p[256:] < 1).all()


@pytest.mark.gpu
def test_side_stream():
    from gfd.optim import Adam
    a, b = make([50000], torch.float32), make([50000], torch.float32)
    one, two = Adam(a, lr=0.1), Adam(b, lr=0.1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        one.step()
        with torch.cuda.stream(side):
            two.step()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a[0], b[0])


@pytest.mark.gpu
def test_refused_on_the_device():
    from gfd.optim import Adam
    p, q = make([40, 30], torch.float32)
    with pytest.raises(ValueError, match="share memory"):
        twice = p.detach()[:10].requires_grad_()
        twice.grad = torch.zeros(10, device=DEV)
        Adam([p, twice]).step()
    with pytest.raises(ValueError, match="dense in memory"):
        Adam([torch.zeros((4, 8), device=DEV)[:, :3].requires_grad_()])
    opt = Adam([p])
    opt.step()
    p.data = torch.zeros(60, device=DEV)
    p.grad = torch.zeros(60, device=DEV)
    with pytest.raises(RuntimeError, match="size"):
        opt.step()
    q.grad = torch.sparse_coo_tensor(torch.tensor([[1]]), torch.tensor([1.0]), (30,)).to(DEV)
    with pytest.raises(RuntimeError, match="dense"):
        Adam([q]).step()
    r = torch.zeros(4, device=DEV, requires_grad=True)
    r.grad = torch.zeros(4, device=DEV)
    with pytest.raises(RuntimeError, match="lr is on"):
        Adam([r], lr=torch.tensor(0.1)).step()


def test_refused_without_a_device():
    from gfd.optim import Adam, AdamW
    p = torch.zeros(4, requires_grad=True)
    p.grad = torch.ones(4)
    with pytest.raises(RuntimeError, match="HIP device"):
        Adam([p]).step()
    for bad in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1e-8),
                dict(weight_decay=-1.0), dict(state_bits=16), dict(seed=-1), dict(lr=float("nan")),
                dict(lr=torch.zeros(2))):
        with pytest.raises(ValueError):
            AdamW([p], **bad)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        Adam([p.detach().double().requires_grad_()])
    assert AdamW([p]).param_groups[0]["weight_decay"] == 1e-2
    assert Adam([p]).param_groups[0]["weight_decay"] == 0.0


def test_c_argument_errors():
    import ctypes as ct

    import numpy as np
    from gfd import _lib
    lib = _lib.load()

    def step(rows=((256, 256, 8, 0, 0),), n=None, dtype=0, bits=32, m=256, v=256, ms=None, vs=None, count=256,
             b1=0.9, eps=1e-8, ticket=256):
        table = np.array(rows, dtype=np.int64)
        return lib.gfd_adam_step(table.ctypes.data_as(ct.c_void_p), len(rows) if n is None else n, dtype, bits, m,
                                 v, ms, vs, count, 1e-3, None, b1, 0.999, eps, 0.0, 0, 0, ticket, None)
    assert step(n=0) == 0 and step(n=-1) == 1
    assert step(dtype=3) == 1 and step(bits=16) == 5 and step(bits=8) == 1
    assert step(m=None) == 1 and step(v=264) == 1 and step(count=None) == 1 and step(ticket=None) == 1
    assert step(b1=1.0) == 1 and step(eps=-1.0) == 1
    for bad in ((0, 256, 8, 0, 0), (256, 0, 8, 0, 0), (256, 256, -1, 0, 0), (256, 256, 8, 100, 0),
                (256, 256, 8, 0, -1), (257, 256, 8, 0, 0)):
        assert step(rows=(bad,)) == 1, bad


class _Written:
    """The library's calls in the place of a launch: what the step's Python does without a GPU."""

    def __init__(self):
        self.calls = []

    def call(self, name, *args):
        self.calls.append(name)

    def call_on(self, device, name, *args):
        self.calls.append(name)

    def gfd_gat_packed_size(self, *shape):
        return 64


def _on_the_host(monkeypatch, params, **kw):
    """An Adam over CPU parameters whose states are there and whose launches do nothing."""
    import types

    from gfd import _lib, optim
    calls = _Written()
    for name in ("call", "call_on"):
        monkeypatch.setattr(_lib, name, getattr(calls, name))
    monkeypatch.setattr(_lib, "load", lambda: calls)
    monkeypatch.setattr(_lib, "stream_handle", lambda device=None: 0)
    opt = optim.Adam(params, **kw)
    f = opt._buffers(params, 32, torch.device("cpu"))
    f["device"] = types.SimpleNamespace(index=-1)
    opt._flat[0] = f
    for i, p in enumerate(params):
        opt.state[p] = opt._views(f, i, p)
    return opt, calls


@pytest.mark.parametrize("missing", [False, True])
def test_a_step_raises_the_versions_of_what_it_writes(monkeypatch, missing):
    """What is derived from a parameter by its version (a layer's packed weights) is made again
    after a step, and a backward pass through an overwritten parameter is refused, as after
    torch's optimizers."""
    from gfd import fused
    from gfd import nn as gnn
    conv = gnn.GATConv(16, 64, heads=8, concat=False)
    params = list(conv.parameters())
    opt, calls = _on_the_host(monkeypatch, params)
    packed, _ = fused.eval_weights(conv, None, torch.device("cpu"))
    for p in params:
        p.grad = torch.ones_like(p)
    if missing:
        params[0].grad = None
    versions = [p._version for p in params]
    moments = opt.state[params[1]]["exp_avg"]._version
    loss = (params[1] * params[1]).sum()
    opt.step()
    assert calls.calls.count("gfd_adam_step") == 1
    assert [p._version - v for p, v in zip(params, versions)] == [0 if missing else 1] + [1] * (len(params) - 1)
    assert opt.state[params[1]]["exp_avg"]._version > moments
    assert fused.eval_weights(conv, None, torch.device("cpu"))[0] is not packed
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_mark_stepped_raises_the_versions(monkeypatch):
    """What a program calls after replays of a captured step, which raise none."""
    p, q = torch.zeros(5, requires_grad=True), torch.zeros(7, requires_grad=True)
    p.grad = torch.ones(5)
    opt, calls = _on_the_host(monkeypatch, [p, q])
    versions = p._version, opt.flat_state()["exp_avg"]._version
    opt.mark_stepped()
    assert p._version > versions[0] and opt.flat_state()["exp_avg"]._version > versions[1] and not calls.calls


@pytest.mark.gpu
def test_a_backward_pass_through_a_stepped_parameter_is_refused():
    from gfd.optim import Adam
    p, = make([300], torch.float32)
    loss = (p * p).sum()
    Adam([p]).step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_a_load_fills_the_states_where_they_are(monkeypatch):
    """A captured step holds their addresses, and that of a tensor lr; one that is refused
    changes neither."""
    params = [torch.zeros(300, requires_grad=True), torch.zeros((7, 5), requires_grad=True)]
    lr = torch.tensor(0.5)
    opt, _ = _on_the_host(monkeypatch, params, lr=lr)
    for k, t in opt.flat_state().items():
        t.copy_(torch.arange(t.numel()))
    saved = copy.deepcopy(opt.state_dict())
    saved["param_groups"][0]["lr"].fill_(0.25)
    del saved["state"][1]
    where = {k: t.data_ptr() for k, t in opt.flat_state().items()}
    for t in opt.flat_state().values():
        t.fill_(9)
    bad = copy.deepcopy(saved)
    bad["state"][0]["exp_avg_sq"] = torch.zeros(3)
    with pytest.raises(ValueError, match="exp_avg_sq"):
        opt.load_state_dict(bad)
    assert lr == 0.5 and all((t == 9).all() for t in opt.flat_state().values())
    for _ in range(2):
        opt.load_state_dict(saved)
        assert {k: t.data_ptr() for k, t in opt.flat_state().items()} == where
        assert opt.param_groups[0]["lr"] is lr and lr == 0.25
        for name in ("exp_avg", "exp_avg_sq"):
            s = [opt.state[p][name] for p in params]
            assert torch.equal(s[0], torch.arange(300.0)) and not s[1].any() and s[1].shape == (7, 5)
        assert opt.flat_state()["step"].tolist() == [0, 0]
        opt.state[params[1]]["exp_avg"].fill_(3.0)
    saved["param_groups"][0]["lr"] = 0.125          # a number goes into the tensor
    opt.load_state_dict(saved)
    assert opt.param_groups[0]["lr"] is lr and lr == 0.125


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_replays_go_on_from_a_loaded_state(bits):
    from gfd.optim import AdamW

    def fresh():
        params = make([5000, (33, 7)], torch.float32)
        return params, AdamW(params, lr=torch.tensor(0.1, device=DEV), state_bits=bits, seed=3)

    (a, captured), (b, eager) = fresh(), fresh()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        captured.step()
    torch.cuda.current_stream().wait_stream(side)
    eager.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured.step()
    saved = copy.deepcopy(eager.state_dict())
    saved["param_groups"][0]["lr"].fill_(0.02)
    saved["state"][0]["step"] += 5
    for _ in range(3):
        captured.load_state_dict(saved)
        eager.load_state_dict(saved)
        torch.full((20000,), float("nan"), device=DEV)     # memory that a load would have given back
        for _ in range(2):
            graph.replay()
            eager.step()
        torch.cuda.synchronize()
        for p, q in zip(a, b):
            assert torch.equal(p, q)
            for k, t in captured.state[p].items():
                assert torch.equal(t.float(), eager.state[q][k].float()), k
    assert eager.state[b[0]]["step"].item() == 8 and torch.equal(eager.param_groups[0]["lr"],
                                                                 captured.param_groups[0]["lr"])


@pytest.mark.gpu
def test_a_load_with_other_bits_makes_the_states_anew():
    from gfd.optim import Adam
    p, = make([700], torch.float32)
    opt = Adam([p], lr=0.1)
    opt.step()
    q, = make([700], torch.float32)
    other = Adam([q], lr=0.1, state_bits=8)
    other.step()
    opt.load_state_dict(other.state_dict())
    assert opt.state[p]["exp_avg"].dtype == torch.float8_e4m3fn
    with torch.no_grad():
        p.copy_(q)
    opt.step()
    other.step()
    assert torch.equal(p, q)


def test_parameters_without_elements_have_a_buffer():
    """The library takes no null pointer for the states."""
    from gfd.optim import Adam
    for bits in (32, 8):
        f = Adam._buffers([torch.zeros(0), torch.zeros(0, 4)], bits, torch.device("cpu"))
        assert all(t.numel() and t.data_ptr() for t in f.values() if isinstance(t, torch.Tensor))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_group_without_elements_steps(bits):
    from gfd.optim import Adam
    p, q = make([0, (0, 3)], torch.float32)
    r, = make([300], torch.float32)
    before = r.detach().clone()
    opt = Adam([{"params": [p, q]}, {"params": [r]}], lr=0.1, state_bits=bits)
    for _ in range(2):
        opt.step()
    assert opt.state[p]["step"].item() == 2 and opt.state[q]["exp_avg"].shape == (0, 3)
    assert not torch.equal(r, before)
    opt.load_state_dict(copy.deepcopy(opt.state_dict()))
    opt.step()
    assert opt.state[q]["step"].item() == 3


def test_a_parameter_that_changes_after_its_states_were_made(monkeypatch):
    """Other strides would take other elements' moments, or memory that is not the parameter's."""
    p = torch.zeros((4, 6), requires_grad=True)
    q = torch.zeros((6, 4)).t().requires_grad_()
    p.grad, q.grad = torch.ones(4, 6), torch.ones(4, 6)
    opt, calls = _on_the_host(monkeypatch, [p, q])
    opt.step()
    assert calls.calls == ["gfd_adam_step"]
    for t, data in ((p, torch.zeros((6, 4)).t()), (p, torch.zeros((4, 12))[:, ::2]), (q, torch.zeros((4, 6))),
                    (q, torch.zeros((6, 8)).t()[:4])):
        was, t.data = t.data, data
        with pytest.raises(RuntimeError, match="strides"):
            opt.step()
        t.data = was
    for t in (p, q):
        t.data, t.grad = t.data.double(), t.grad.double()
    with pytest.raises(RuntimeError, match="type"):
        opt.step()
    assert calls.calls == ["gfd_adam_step"]


def test_the_options_of_torch():
    """torch's constructor calls: what changes the rule is refused, what chooses an implementation
    taken."""
    from gfd.optim import Adam, AdamW
    p = torch.zeros(4, requires_grad=True)
    for cls in (Adam, AdamW):
        opt = cls([p], 1e-2, (0.8, 0.9), 1e-6, 0.1, False, foreach=True, maximize=False, capturable=True,
                  differentiable=False, fused=None, state_bits=8, seed=3)
        group = opt.param_groups[0]
        assert (group["lr"], group["weight_decay"], group["state_bits"], group["seed"]) == (1e-2, 0.1, 8, 3)
        for name in ("amsgrad", "maximize", "differentiable"):
            with pytest.raises(NotImplementedError, match=name):
                cls([p], **{name: True})
            with pytest.raises(NotImplementedError, match=name):
                cls([{"params": [p], name: True}])
        with pytest.raises(TypeError):
            cls([p], decay=1.0)


def test_a_load_after_the_states_were_dropped(monkeypatch):
    """``opt.state`` cleared by hand, and a group of no parameters beside: the load fills the
    buffers, and the views are there again."""
    p = torch.zeros(300, requires_grad=True)
    opt, _ = _on_the_host(monkeypatch, [p])
    opt.flat_state()["exp_avg"].fill_(2.0)
    saved = copy.deepcopy(opt.state_dict())
    opt.flat_state()["exp_avg"].zero_()
    opt.state.clear()
    opt.load_state_dict(saved)
    assert (opt.state[p]["exp_avg"] == 2.0).all()
    opt.param_groups.append(dict(opt.param_groups[0], params=[]))
    opt.mark_stepped()
