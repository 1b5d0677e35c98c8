"""The operators of a training step together: a GAT with group norms scored by
class log probabilities with an entropy bonus, its backward, and an Adam / AdamW
step -- against the fp64 oracle's model, and captured into a graph."""
import pytest
import torch
import torch.nn.functional as F

from _util import assert_close, assert_close_scaled

DEV = "cuda"
N, E, WIDTH, CLASSES = 1500, 6000, 37, 5


def _problem(seed=0):
    g = torch.Generator().manual_seed(seed)
    ei = torch.randint(N, (2, E), generator=g)
    x = torch.randn(N, WIDTH, generator=g)
    y = torch.randint(CLASSES, (N,), generator=g)
    y[torch.rand(N, generator=g) < 0.3] = -1
    return ei, x, y


def _model(kind="GAT", **kw):
    from gfd import models
    torch.manual_seed(2)
    m = getattr(models, kind)(WIDTH, 64, CLASSES, num_layers=2, dropout=0.0, norm="group", num_groups=8, **kw)
    with torch.no_grad():
        for norm in m.group_norms:
            norm.weight.uniform_(0.5, 1.5)
            norm.bias.uniform_(-0.2, 0.2)
    return m


def _oracle_loss(m, ei, x, y):
    """The same model and loss in fp64 from the oracle's GATConv; parameters by name."""
    from oracle import gatconv_ref as ref
    p = {k: v.detach().cpu().double().requires_grad_() for k, v in m.named_parameters()}
    h = x.double()
    for li in range(2):
        c = f"gat_layers.{li}."
        z = ref.gatconv_forward(h, ei, p[c + "lin_src.weight"], p[c + "att_src"], p[c + "att_dst"], p[c + "bias"])
        z = F.group_norm(z, 8, p[f"group_norms.{li}.weight"], p[f"group_norms.{li}.bias"]).relu()
        h = h + z if h.shape == z.shape else z
    logits = h @ p["out.weight"].t() + p["out.bias"]
    logp = torch.log_softmax(logits, 1)
    known = y >= 0
    loss = -logp[known].gather(1, y[known][:, None]).sum() / known.sum()
    entropy = -(logp.exp() * logp).sum(1)
    return loss - 0.05 * entropy.mean(), p, logits.detach()


def _loss(m, ei, x, y):
    r = m.log_probs(x, ei, y, top=2)
    return -r.log_prob.sum() / (y >= 0).sum() - 0.05 * r.entropy.mean(), r


@pytest.mark.gpu
def test_step_against_the_oracle():
    from gfd.optim import AdamW
    ei, x, y = _problem()
    m = _model().to(DEV).train()
    loss, r = _loss(m, ei.to(DEV), x.to(DEV), y.to(DEV))
    loss.backward()
    ref, p, logits = _oracle_loss(m, ei, x, y)
    ref.backward()
    assert abs(loss.item() - ref.item()) <= 1e-5 * abs(ref.item())
    sure = logits.sort(1, descending=True).values[:, :3].diff(dim=1).abs().min(1).values > 1e-3
    assert torch.equal(r.top_classes.cpu()[sure], logits.topk(2, 1).indices[sure])
    for k, v in m.named_parameters():
        # a gradient's fp32 sums against fp64: 2e-4 of its largest, and what is 0 up to noise
        assert_close_scaled(v.grad, p[k].grad, rtol=2e-4, atol=1e-7, what=k)
    # the step itself, on the device's own gradients
    theirs = [v.detach().cpu().double().requires_grad_() for v in m.parameters()]
    for a, v in zip(theirs, m.parameters()):
        a.grad = v.grad.cpu().double()
    opt, topt = AdamW(m.parameters(), lr=1e-2), torch.optim.AdamW(theirs, lr=1e-2)
    opt.step()
    topt.step()
    for a, v in zip(theirs, m.parameters()):
        # 16 U of the update (lr) and of the parameter, and its rounding
        assert (v.detach().cpu().double() - a.detach()).abs().max() <= 20 * 2.0 ** -24 * (1e-2 + a.abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["GAT", "TemporalGNN"])
@pytest.mark.parametrize("bits", [32, 8])
def test_training_runs(kind, bits):
    from gfd.optim import Adam
    ei, x, y = (t.to(DEV) for t in _problem())
    m = _model(kind).to(DEV).train()
    opt = Adam(m.parameters(), lr=1e-3, weight_decay=5e-4, state_bits=bits)
    before = [p.detach().clone() for p in m.parameters()]
    for _ in range(3):
        opt.zero_grad()
        loss, _ = _loss(m, ei, x, y)
        loss.backward()
        opt.step()
    assert torch.isfinite(loss)
    for a, p in zip(before, m.parameters()):
        assert p.isfinite().all() and (p.grad is None or not torch.equal(a, p) or not p.grad.any())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["GAT", "TemporalGNN"])
def test_snapshots_in_training_equal_their_own_passes(kind):
    """A node's statistics are its own row's: the step-by-step graphs of a temporal graph and
    the whole give the same in training mode, which batch statistics do not."""
    ei, x, _ = _problem()
    step = torch.arange(N) * 3 // N
    ei = ei[:, step[ei[0]] == step[ei[1]]]
    m = _model(kind).to(DEV).train()
    whole = m(x.to(DEV), ei.to(DEV))
    whole = whole[0] if isinstance(whole, tuple) else whole
    for s in range(3):
        at = (step == s).nonzero()[:, 0]
        sub = ei[:, step[ei[0]] == s] - at[0]
        part = m(x[at].to(DEV), sub.contiguous().to(DEV))
        part = part[0] if isinstance(part, tuple) else part
        assert_close(part, whole[at.to(DEV)].detach(), what=f"step {s}")


@pytest.mark.gpu
def test_eval_equals_training_mode_and_no_grad():
    ei, x, y = (t.to(DEV) for t in _problem())
    m = _model().to(DEV)
    a = m.train()(x, ei)
    with torch.no_grad():
        b = m.eval()(x, ei)
        r = m.log_probs(x, ei, y, top=1)
    assert_close(b, a.detach(), what="eval")
    assert torch.equal(r.top_classes[:, 0], b.argmax(1))


@pytest.mark.gpu
def test_rows_scores_and_step_captured_together():
    """A head over frozen features: norm, scores, gradients and step in one graph, replayed
    with eager steps of a second copy between."""
    from gfd.fused import class_log_probs, group_norm
    from gfd.optim import AdamW
    gen = torch.Generator().manual_seed(5)
    x = torch.randn(900, 64, generator=gen).to(DEV)
    y = torch.randint(-1, CLASSES, (900,), generator=gen).to(DEV)
    start = [torch.randn(s, generator=gen).to(DEV) * 0.1 for s in ((64,), (64,), (CLASSES, 64))]

    def make():
        params = [p.clone().requires_grad_() for p in start]
        opt = AdamW(params, lr=1e-2, state_bits=8, seed=4)
        for p in params:
            p.grad = torch.zeros_like(p)

        def step():
            leaves = [p.detach().requires_grad_() for p in params]
            h = group_norm(x, 8, leaves[0] + 1, leaves[1], act="silu")
            r = class_log_probs(h @ leaves[2].t(), y)
            loss = -r.log_prob.mean() - 0.01 * r.entropy.mean()
            for p, g in zip(params, torch.autograd.grad(loss, leaves)):
                p.grad.copy_(g)
            opt.step()
        return params, step

    (a, captured), (b, eager) = make(), make()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        captured()
    torch.cuda.current_stream().wait_stream(side)
    eager()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured()
    for _ in range(3):
        graph.replay()
        eager()
        torch.cuda.synchronize()
        for p, q in zip(a, b):
            # the head's product and the means are the library's: their order may differ in a graph
            assert_close_scaled(p, q, rtol=1e-3)


def _sharded_rank(rank, world, path, q):
    import torch.distributed as dist
    from gfd import dist as gdist, graph as ggraph
    dist.init_process_group("gloo", init_method=f"file://{path}", rank=rank, world_size=world)
    try:
        ei, x, y = _problem()
        m = _model().to(DEV).train()
        g = ggraph.csr_from_coo(ei.to(DEV), N)
        spec = gdist.ShardSpec(g.rowptr.long(), rank, world, "cost")
        lo, hi = spec.dst_lo, spec.dst_hi
        rp = g.rowptr.long()
        plan = gdist.HaloPlan.create(g.col[int(rp[lo]):int(rp[hi])], spec)
        logits = gdist.gat_forward_sharded_train(m, x.to(DEV), gdist.local_graph(g, lo, hi), plan, N)
        from gfd.fused import class_log_probs
        r = class_log_probs(logits, y[lo:hi].to(DEV))
        (-r.log_prob.sum() / int((y >= 0).sum()) - 0.05 * r.entropy.sum() / N).backward()
        gdist.all_reduce_grads(list(m.parameters()))
        if rank == 0:
            q.put({k: p.grad.cpu().numpy() for k, p in m.named_parameters()})
        dist.barrier()
    finally:
        dist.destroy_process_group()


@pytest.mark.gpu
def test_sharded_step_needs_no_exchange_for_the_norm():
    import torch.multiprocessing as mp
    from test_dist_cpu import _store_path
    ctx = mp.get_context("spawn")
    q, path = ctx.Queue(), _store_path()
    procs = [ctx.Process(target=_sharded_rank, args=(r, 2, path, q)) for r in range(2)]
    for p in procs:
        p.start()
    got = q.get(timeout=100)
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    ei, x, y = _problem()
    ref, p, _ = _oracle_loss(_model(), ei, x, y)
    ref.backward()
    for k, g in got.items():
        assert_close_scaled(torch.from_numpy(g), p[k].grad, rtol=2e-4, atol=1e-7, what=k)


def test_norm_argument_and_state_dict_keys():
    from gfd.models import GAT, TemporalGNN
    with pytest.raises(ValueError, match="norm must be"):
        GAT(8, 64, 2, norm="layer")
    with pytest.raises(ValueError, match="divisible"):
        GAT(8, 64, 2, norm="group", num_groups=7)
    assert not any("group_norms" in k for k in GAT(8, 64, 2).state_dict())
    keys = TemporalGNN(8, 64, 2, norm="group").state_dict()
    assert "group_norms.1.weight" in keys and not any("batch_norms" in k for k in keys)


def test_sharded_inference_refuses_group_norms():
    from gfd import dist as gdist
    m = _model().eval()
    with torch.no_grad(), pytest.raises(NotImplementedError, match="norm='group'"):
        gdist.model_forward_sharded(m, None, None, None)


def test_stream_of_any_form_of_a_device(monkeypatch):
    """A device by its name, as an object with or without an index, or none at all."""
    from gfd import _lib

    class Stream:
        cuda_stream = 7

    seen = []
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: seen.append(device) or Stream)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 100 + int(index), raising=False)
    for device in ("cuda", "cuda:0", torch.device("cuda"), None):
        assert _lib.stream_handle(device) == 7 and seen.pop() == device
    assert _lib.stream_handle(torch.device("cuda", 2)) == 102 and not seen


@pytest.mark.gpu
@pytest.mark.parametrize("norm", ["batch", "group"])
@pytest.mark.parametrize("kind", ["GAT", "TemporalGNN"])
def test_evaluation_follows_a_step(kind, norm):
    """evaluate, step, evaluate: the second evaluation is a fresh model's of the same state."""
    from gfd import models
    from gfd.optim import AdamW
    ei, x, y = (t.to(DEV) for t in _problem())

    def make():
        torch.manual_seed(3)
        return getattr(models, kind)(WIDTH, 64, CLASSES, num_layers=2, dropout=0.0, norm=norm).to(DEV)

    def evaluate(m):
        with torch.no_grad():
            return m.eval().log_probs(x, ei, y, top=2)

    m = make()
    opt = AdamW(m.parameters(), lr=1e-2)
    before = evaluate(m)
    for _ in range(2):
        opt.zero_grad()
        loss, _ = _loss(m.train(), ei, x, y)
        loss.backward()
        opt.step()
        after, fresh = evaluate(m), make()
        fresh.load_state_dict(m.state_dict())
        for a, b in zip(after, evaluate(fresh)):
            assert torch.equal(a, b)
        assert not torch.equal(after.entropy, before.entropy)


@pytest.mark.gpu
def test_evaluation_follows_replays_of_a_captured_step():
    from gfd.optim import AdamW
    ei, x, y = (t.to(DEV) for t in _problem())
    m, fresh = _model().to(DEV), _model().to(DEV)
    opt = AdamW(m.parameters(), lr=1e-2)
    for p in m.parameters():
        p.grad = torch.full_like(p, 0.1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        opt.step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    with torch.no_grad():
        for _ in range(2):
            m.eval()(x, ei)
            graph.replay()
            opt.mark_stepped()
            fresh.load_state_dict(m.state_dict())
            assert torch.equal(m.eval()(x, ei), fresh.eval()(x, ei))


@pytest.mark.parametrize("place", range(3))
def test_a_tangent_is_seen(place):
    """Of any of the inputs, with and without gradients, and only while its level is open."""
    from torch.autograd import forward_ad

    from gfd.fused import _needs_grad
    inputs = [torch.ones(4), None, torch.ones(4)]
    with forward_ad.dual_level():
        assert not _needs_grad(*inputs)
        if inputs[place] is not None:
            inputs[place] = forward_ad.make_dual(inputs[place], torch.ones(4))
        assert _needs_grad(*inputs) == (inputs[place] is not None)
        with torch.no_grad():
            assert _needs_grad(*inputs) == (inputs[place] is not None)
    assert not _needs_grad(*inputs) and not _needs_grad(None)


@pytest.mark.gpu
def test_forward_mode_is_refused():
    """Neither operator has a forward-mode derivative: an input with a tangent is an error, not a
    result without one."""
    from torch.autograd import forward_ad

    from gfd.fused import class_log_probs, group_norm
    x, w = torch.randn(5, 8, device=DEV), torch.ones(8, device=DEV)
    with forward_ad.dual_level():
        d, dw = (forward_ad.make_dual(t, torch.ones_like(t)) for t in (x, w))
        for call in (lambda: group_norm(d, 2), lambda: group_norm(d[None], 2, w), lambda: group_norm(x, 2, dw),
                     lambda: group_norm(x, 2, w, dw), lambda: class_log_probs(d, top=1),
                     lambda: class_log_probs(d[0])):
            with pytest.raises(NotImplementedError):
                call()
        assert forward_ad.unpack_dual(group_norm(x, 2)).tangent is None


class _Calls:
    """The library's calls in the place of their launches."""

    def __init__(self):
        self.args = {}

    def call_on(self, device, name, *args):
        self.args[name] = args

    def gfd_group_norm_workspace_size(self, *shape):
        return 16

    def gfd_class_logp_workspace_size(self, *shape):
        return 0


def _elsewhere(t):
    """A copy with other strides: of rows at a larger pitch."""
    if t.dim() != 2:
        return torch.stack((t, t), -1)[..., 0] if t.dim() == 1 else t.clone()
    return torch.cat((t, t[:, :1]), 1)[:, :-1]


def test_saved_tensors_that_come_back_elsewhere(monkeypatch):
    """Saved-tensor hooks (offloading, checkpoints) hand the backward copies: their addresses and
    strides go to the library, not those of the forward's tensors."""
    from gfd import _lib, fused
    calls = _Calls()
    monkeypatch.setattr(_lib, "call_on", calls.call_on)
    monkeypatch.setattr(_lib, "load", lambda: calls)
    monkeypatch.setattr(_lib, "stream_handle", lambda device=None: 0)
    came = []

    def unpack(t):
        came.append(_elsewhere(t))
        return came[-1]

    x = torch.randn(40, 12)[:, 2:10].requires_grad_()
    w, ptr = torch.ones(8, requires_grad=True), torch.tensor([0, 3, 40])
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        y = fused._GroupNorm.apply(x, w, None, ptr, 2, 1e-5, 1)
        y.backward(torch.ones(40, 8))
    a = calls.args["gfd_group_norm_bwd"]
    assert calls.args["gfd_group_norm_fwd"][4] == ptr.data_ptr() != a[4]
    assert a[0] in [t.data_ptr() for t in came if t.stride() == (9, 1)] and a[7:9] == (9, 0)
    assert a[1:4] == (0, 2, 40) and a[5:7] == (8, 2) and a[9] != w.data_ptr()
    came.clear()
    x.grad = None
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        logp, entropy, _, _ = fused._ClassLogProbs.apply(x, torch.zeros(40, dtype=torch.int64), 2, -1)
        (logp.sum() + entropy.sum()).backward()
    f, a = calls.args["gfd_class_logp_fwd"], calls.args["gfd_class_logp_bwd"]
    assert f[:5] == (x.data_ptr(), 0, 40, 8, 12) and a[1:5] == (0, 40, 8, 9)
    assert a[0] in [t.data_ptr() for t in came if t.stride() == (9, 1)] and a[5] != f[5]


@pytest.mark.gpu
def test_offloaded_and_checkpointed_passes_give_the_same_gradients():
    from torch.utils.checkpoint import checkpoint

    from gfd.fused import class_log_probs, group_norm
    base = torch.randn(300, 70, device=DEV)
    ptr = torch.tensor([0, 0, 5, 5, 200, 0, 290, 0], device=DEV)[::2]     # a copy of it is taken
    t = torch.randint(-1, 64, (300,), device=DEV)
    w = torch.rand(64, device=DEV)

    def passes(x, w):
        h = group_norm(x, 8, w, act="silu", ptr=ptr)
        r = class_log_probs(group_norm(h, 8) * 2, t, top=3)
        s = class_log_probs(x, t, top=1)
        return r.log_prob.sum() + r.entropy.sum() + s.log_prob.sum() + 0.5 * s.top_log_probs.sum()

    def grads(run):
        leaf, lw = base.clone().requires_grad_(), w.clone().requires_grad_()
        return torch.autograd.grad(run(leaf[:, 3:67], lw), (leaf, lw))

    def offloaded(x, w):
        with torch.autograd.graph.save_on_cpu():
            return passes(x, w)

    want = grads(passes)
    for run in (offloaded, lambda x, w: checkpoint(passes, x, w, use_reentrant=False)):
        for a, b in zip(grads(run), want):
            # another alignment is another order of a row's fp32 sums: 48 roundings, for each of
            # the three passes
            assert_close_scaled(a, b, rtol=3 * 48 * 2.0 ** -24)


@pytest.mark.gpu
def test_evaluation_follows_new_running_statistics():
    """A training-mode pass without a step between two evaluations."""
    from gfd import models
    ei, x, _ = (t.to(DEV) for t in _problem())

    def make():
        torch.manual_seed(3)
        return models.GAT(WIDTH, 64, 1, num_layers=2, dropout=0.0).to(DEV)

    m, fresh = make(), make()
    with torch.no_grad():
        before = m.eval()(x, ei)
        m.train()(x * 3, ei)
        fresh.load_state_dict(m.state_dict())
        after = m.eval()(x, ei)
        assert torch.equal(after, fresh.eval()(x, ei)) and not torch.equal(after, before)
