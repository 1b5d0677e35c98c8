"""Fused inference paths of the reference model bodies.

* ``gat_layer`` -- one layer of /root/reference/src/models/gat.py:79-91 (and
  tgn.py:93-105) in eval mode: GATConv -> BatchNorm1d(running stats) -> ReLU
  -> dropout (identity) -> residual, as ONE call of ``gfd_gat_fwd_ep``: the
  BatchNorm folds into a per-channel affine applied where the tile kernels
  store each output row, so the layer output is written once (the unfused
  path writes the GATConv output, then BN, ReLU and the residual add each
  read and write [N, 64] again).
* ``gru_head`` -- the TemporalGNN head (tgn.py:108-111): GRUCell(h, h0) +
  Linear in one kernel (``gfd_gru_head``); ``tgn_head_train`` -- the same
  head in training mode, forward and backward on the device
  (``gfd_gru_head_bwd`` + ``gfd_atb``).

* ``train_body`` -- the same layer body in training mode after the GATConv:
  residual + dropout(relu(BatchNorm1d(y))) with batch statistics, as one
  autograd Function over ``gfd_bn_relu_fwd`` / ``gfd_bn_relu_bwd`` (two
  passes over y each way instead of ATen's BN / relu / dropout / add chain
  and its saved intermediates; only y and two [64] vectors are kept).

* ``group_norm`` -- group norm with an activation over node rows (dense or
  ragged segments), forward and backward (``gfd_group_norm_fwd`` / ``_bwd``):
  statistics that stay inside a node, a snapshot or a sampled subgraph.
* ``class_log_probs`` -- log probabilities of given classes with entropy and
  top alternatives from a classification head's logits, forward and backward
  (``gfd_class_logp_fwd`` / ``_bwd``).

``gat_layer`` and ``gru_head`` are inference-only: they refuse tensors that
require grad (gfd.models takes ``GATConv`` + ``train_body`` then).
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from .graph import CSRGraph, _ws, get_graph
from .nn import SUPPORTED_CHANNELS, SUPPORTED_HEADS, _rows

H, C = SUPPORTED_HEADS, SUPPORTED_CHANNELS


def bn_affine(bn: Optional[torch.nn.BatchNorm1d], device) -> torch.Tensor:
    """[2C] (scale | shift) of an eval-mode BatchNorm1d: y = x * scale + shift
    with scale = gamma / sqrt(running_var + eps), shift = beta - mean * scale
    (identity when ``bn`` is None)."""
    if bn is None:
        return torch.cat([torch.ones(C, device=device), torch.zeros(C, device=device)])
    if not bn.track_running_stats or bn.running_var is None:
        raise NotImplementedError("fused BatchNorm needs running statistics (eval mode)")
    scale = torch.rsqrt(bn.running_var.float() + bn.eps)
    if bn.affine:
        scale = scale * bn.weight.float()
    shift = -bn.running_mean.float() * scale
    if bn.affine:
        shift = shift + bn.bias.float()
    return torch.cat([scale, shift]).contiguous()


def head_foldable(head, width: int, conv=None) -> bool:
    """The model head the store can fold (gfd_epilogue.head_*): Linear(64, 1)
    in fp32 after a layer whose input width takes the plan-scheduled kernels
    (F <= 168) and, when ``conv`` (the last GATConv) is given, whose attention
    slope those kernels take (leaky01: negative_slope in [0, 1]; others go to
    the head-less k_fused path, which cannot fold the head)."""
    if conv is not None and not (0.0 <= float(conv.negative_slope) <= 1.0):
        return False
    return (head is not None and head.in_features == C and head.out_features == 1 and
            head.weight.dtype == torch.float32 and head.weight.is_cuda and width <= 168 and
            (head.bias is None or head.bias.dtype == torch.float32))


def check_params(conv, bn, device) -> None:
    """The checks GATConvFunction.forward makes on the layer's tensors, for the
    packed-weights inference paths (eval_conv, gat_layer): their pointers go
    to the kernels on x's stream, so a parameter left on the CPU, on another
    GPU or in another dtype must raise here, not fault or read garbage there
    (ADVICE r5)."""
    from .nn import _check_tensor
    _check_tensor("lin_src.weight", conv.lin_src.weight, device)
    _check_tensor("att_src", conv.att_src, device)
    _check_tensor("att_dst", conv.att_dst, device)
    if conv.bias is not None:
        _check_tensor("bias", conv.bias, device)
    if bn is not None:
        for n in ("running_mean", "running_var", "weight", "bias"):
            t = getattr(bn, n, None)
            if t is not None:
                _check_tensor(f"BatchNorm {n}", t, device)


def eval_weights(conv, bn, device) -> Tuple[torch.Tensor, torch.Tensor]:
    """(packed weights, BatchNorm scale | shift) of an inference layer, rebuilt
    only when a tensor they derive from changed: the cache on ``conv`` holds
    each source tensor, its version counter and storage address, so a replaced
    parameter (a new object), an in-place update (optimizer step,
    load_state_dict) or new storage (``.to(device)``) rebuilds it, while
    evaluation over many batches (evaluate.py:73-98) packs once."""
    srcs = [conv.lin_src.weight, conv.att_src, conv.att_dst]
    if bn is not None:
        srcs += [bn.running_mean, bn.running_var]
        if bn.affine:
            srcs += [bn.weight, bn.bias]
    # (object, version, storage address): a module moved to another device or
    # given new .data keeps its parameter objects but not their storage
    key = [(t, t._version, t.data_ptr()) for t in srcs] + [bn.eps if bn is not None else None,
                                                             bn, str(device)]
    c = conv.__dict__.get("_gfd_eval")
    if c is not None and len(c[0]) == len(key) and all(
            (a[0] is b[0] and a[1:] == b[1:]) if isinstance(a, tuple) else a is b or a == b
            for a, b in zip(c[0], key)):
        return c[1], c[2]
    W = conv.lin_src.weight.detach().contiguous()
    F = W.size(1)
    lib = _lib.load()
    packed = torch.empty(lib.gfd_gat_packed_size(F, H, C), dtype=torch.uint8, device=device)
    _lib.call("gfd_gat_pack_weights", W.data_ptr(),
              conv.att_src.detach().reshape(-1).contiguous().data_ptr(),
              conv.att_dst.detach().reshape(-1).contiguous().data_ptr(), F, H, C,
              packed.data_ptr(), _lib.stream_handle(device))
    ab = bn_affine(bn, device)
    conv.__dict__["_gfd_eval"] = (key, packed, ab)
    return packed, ab


def eval_conv(conv, x: torch.Tensor, edge_index) -> torch.Tensor:
    """``conv(x, edge_index)`` in inference (no autograd, no dropout) with the
    layer's packed weights from ``eval_weights``: the drop-in module's
    ``torch.no_grad()`` forward (gat.py:80 under evaluate.py:73-98)."""
    from .nn import _check_tensor
    dev = x.device
    _check_tensor("x", x, dev, (torch.float32, torch.bfloat16))
    graph = edge_index if isinstance(edge_index, CSRGraph) else get_graph(edge_index, x.size(0))
    if graph.num_nodes != x.size(0):
        raise ValueError(f"graph has {graph.num_nodes} nodes but x has {x.size(0)} rows")
    x = _rows(x)
    N, F = x.shape
    if F != conv.lin_src.weight.size(1):
        raise ValueError(f"x has {F} features, the layer expects {conv.lin_src.weight.size(1)}")
    check_params(conv, None, dev)
    packed, _ = eval_weights(conv, None, dev)
    bias = conv.bias.detach() if conv.bias is not None else None
    plan = graph.plan()
    lib = _lib.load()
    out = torch.empty((N, C), dtype=torch.float32, device=dev)
    ws = _ws(lib.gfd_gat_fwd_workspace_size(N, N, F, H, C, plan.num_hubs, plan.num_chunks), dev)
    _lib.call("gfd_gat_fwd_ep_packed", x.data_ptr(), _lib.x_dtype_code(x), N, F, x.stride(0),
              graph.rowptr.data_ptr(), graph.col.data_ptr(), packed.data_ptr(), _lib.ptr(bias),
              H, C, float(conv.negative_slope), 0.0, 0, plan.cstruct(), None, out.data_ptr(),
              None, None, ws.data_ptr(), ws.numel(), _lib.stream_handle(dev))
    return out


def gat_layer(conv, bn, h: torch.Tensor, edge_index, relu: bool = True,
              residual: bool = False, head=None) -> torch.Tensor:
    """One eval-mode layer body: residual(h) + relu(bn(conv(h, edge_index))).
    ``head`` (Linear(64, 1), see head_foldable): the model head folded into
    the store (gat.py:94) -- returns head(body) [N, 1] and the [N, 64] body
    is never written."""
    if torch.is_grad_enabled() and (h.requires_grad or conv.lin_src.weight.requires_grad):
        raise RuntimeError("gfd.fused.gat_layer is inference-only (use torch.no_grad())")
    dev = h.device
    graph = edge_index if isinstance(edge_index, CSRGraph) else get_graph(edge_index, h.size(0))
    x = _rows(h)
    N, F = x.shape
    bias = conv.bias.detach() if conv.bias is not None else None
    check_params(conv, bn, dev)
    packed, ab = eval_weights(conv, bn, dev)
    res = None
    if residual:
        if F != C:
            raise ValueError("residual needs the layer input width to equal 64")
        # the epilogue adds fp32 rows (gfd_epilogue.residual is float*)
        res = x if x.dtype == torch.float32 else x.float()
    hout = hw = None
    if head is not None:
        if not head_foldable(head, F, conv):
            raise ValueError("gat_layer head: Linear(64, 1) fp32 on the device after a layer the "
                             "plan-scheduled kernels take (head_foldable)")
        hw = head.weight.detach().reshape(-1).contiguous()
        hout = torch.empty((N, 1), dtype=torch.float32, device=dev)
    ep = _lib.GfdEpilogue(ab.data_ptr(), 1 if relu else 0, _lib.ptr(res),
                          res.stride(0) if res is not None else 0, _lib.ptr(hw),
                          _lib.ptr(head.bias.detach() if head is not None and
                                   head.bias is not None else None), _lib.ptr(hout))
    plan = graph.plan()
    lib = _lib.load()
    out = torch.empty((N, C), dtype=torch.float32, device=dev) if hout is None else None
    ws = _ws(lib.gfd_gat_fwd_workspace_size(N, N, F, H, C, plan.num_hubs, plan.num_chunks), dev)
    _lib.call("gfd_gat_fwd_ep_packed", x.data_ptr(), _lib.x_dtype_code(x), N, F, x.stride(0),
              graph.rowptr.data_ptr(), graph.col.data_ptr(), packed.data_ptr(), _lib.ptr(bias),
              H, C, float(conv.negative_slope), 0.0, 0, plan.cstruct(), _lib.ct.byref(ep),
              _lib.ptr(out), None, None, ws.data_ptr(), ws.numel(), _lib.stream_handle(dev))
    return out if hout is None else hout


def gru_head(gru: torch.nn.GRUCell, lin: torch.nn.Linear, h: torch.Tensor,
             h0: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(lin(GRUCell(h, h0)), GRUCell(h, h0)) in one kernel (h0 None = zeros)."""
    if torch.is_grad_enabled() and (h.requires_grad or gru.weight_ih.requires_grad):
        raise RuntimeError("gfd.fused.gru_head is inference-only (use torch.no_grad())")
    if gru.hidden_size != C or gru.input_size != C:
        raise NotImplementedError("gfd gru_head: GRUCell(64, 64)")
    dev = h.device
    x = h.float() if h.dtype != torch.float32 else h      # the kernel reads fp32 rows
    x = x if x.stride(1) == 1 and x.stride(0) % 4 == 0 else x.contiguous()
    if h0 is not None:
        h0 = h0.float() if h0.dtype != torch.float32 else h0
        h0 = h0 if h0.stride(1) == 1 and h0.stride(0) % 4 == 0 else h0.contiguous()
    N = x.size(0)
    O = lin.out_features
    h_new = torch.empty((N, C), dtype=torch.float32, device=dev)
    out = torch.empty((N, O), dtype=torch.float32, device=dev)
    w_ih, w_hh = gru.weight_ih.detach().contiguous(), gru.weight_hh.detach().contiguous()
    b_ih = gru.bias_ih.detach() if gru.bias else None
    b_hh = gru.bias_hh.detach() if gru.bias else None
    w_o = lin.weight.detach().contiguous()
    b_o = lin.bias.detach() if lin.bias is not None else None
    _lib.call("gfd_gru_head", x.data_ptr(), N, C, x.stride(0), w_ih.data_ptr(), _lib.ptr(b_ih),
              w_hh.data_ptr(), _lib.ptr(b_hh), _lib.ptr(h0), h0.stride(0) if h0 is not None else 0,
              w_o.data_ptr(), _lib.ptr(b_o), O, h_new.data_ptr(), out.data_ptr(),
              _lib.stream_handle(dev))
    return out, h_new


class _GRUHeadTrain(torch.autograd.Function):
    """(out, h_new) = (Linear(GRUCell(h, h0)), GRUCell(h, h0)) with both
    directions on the device: forward = gfd_gru_head (the inference kernel:
    gates on fp32 MFMA, nothing but h / h0 / h_new kept), backward =
    gfd_gru_head_bwd (gates recomputed, gate gradients, grad_h / grad_h0) +
    gfd_atb for the six weight / bias gradients (deterministic sums)."""

    @staticmethod
    def forward(ctx, h, h0, w_ih, b_ih, w_hh, b_hh, w_o, b_o):
        dev = h.device
        N = h.size(0)
        O = w_o.size(0)
        h_new = torch.empty((N, C), dtype=torch.float32, device=dev)
        out = torch.empty((N, O), dtype=torch.float32, device=dev)
        _lib.call("gfd_gru_head", h.data_ptr(), N, C, h.stride(0), w_ih.data_ptr(), _lib.ptr(b_ih),
                  w_hh.data_ptr(), _lib.ptr(b_hh), _lib.ptr(h0),
                  h0.stride(0) if h0 is not None else 0, w_o.data_ptr(), _lib.ptr(b_o), O,
                  h_new.data_ptr(), out.data_ptr(), _lib.stream_handle(dev))
        ctx.save_for_backward(h, h0, w_ih, b_ih, w_hh, b_hh, w_o, b_o, h_new)
        return out, h_new

    @staticmethod
    def backward(ctx, g_out, g_hnew):
        h, h0, w_ih, b_ih, w_hh, b_hh, w_o, b_o, h_new = ctx.saved_tensors
        dev = h.device
        N, O = h.size(0), w_o.size(0)
        lib = _lib.load()
        stream = _lib.stream_handle(dev)
        g_out = (g_out if g_out is not None else torch.zeros((N, O), device=dev)).float().contiguous()
        g_hnew = g_hnew.float().contiguous() if g_hnew is not None else None
        grad_h = torch.empty((N, C), dtype=torch.float32, device=dev)
        grad_h0 = torch.empty((N, C), dtype=torch.float32, device=dev) if h0 is not None else None
        gi = torch.empty((N, 3 * C), dtype=torch.float32, device=dev)
        gh = torch.empty_like(gi)
        _lib.call("gfd_gru_head_bwd", h.data_ptr(), N, C, h.stride(0), w_ih.data_ptr(),
                  _lib.ptr(b_ih), w_hh.data_ptr(), _lib.ptr(b_hh), _lib.ptr(h0),
                  h0.stride(0) if h0 is not None else 0, w_o.data_ptr(), O, g_out.data_ptr(),
                  _lib.ptr(g_hnew), grad_h.data_ptr(), _lib.ptr(grad_h0), gi.data_ptr(),
                  gh.data_ptr(), stream)
        ws = _ws(lib.gfd_atb_workspace_size(N, 3 * C), dev)

        def atb(A, m, B):
            wgt = torch.empty((m, C), dtype=torch.float32, device=dev)
            col = torch.empty((m,), dtype=torch.float32, device=dev)
            _lib.call("gfd_atb", A.data_ptr(), A.stride(0), m, _lib.ptr(B),
                      B.stride(0) if B is not None else C, N, wgt.data_ptr(), col.data_ptr(),
                      ws.data_ptr(), ws.numel(), stream)
            return wgt, col

        g_wih, g_bih = atb(gi, 3 * C, h)
        if h0 is not None:
            g_whh, g_bhh = atb(gh, 3 * C, h0)
        else:                                   # h0 = 0: no W_hh product, only b_hh
            g_whh = torch.zeros_like(w_hh)
            g_bhh = atb(gh, 3 * C, h)[1]
        g_wo, g_bo = atb(g_out, O, h_new)
        return (grad_h, grad_h0, g_wih, g_bih if b_ih is not None else None, g_whh,
                g_bhh if b_hh is not None else None, g_wo, g_bo if b_o is not None else None)


def _aligned_rows(t: torch.Tensor) -> torch.Tensor:
    """t itself when its rows are unit-stride, 16-B aligned and at a 16-B
    multiple pitch (what gfd_gru_head / _bwd read as vectors); otherwise a
    fresh contiguous copy -- also for a contiguous view at a misaligned offset,
    which .contiguous() would return unchanged."""
    if t.stride(1) == 1 and t.stride(0) % 4 == 0 and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def tgn_head_train(gru: torch.nn.GRUCell, lin: torch.nn.Linear, h: torch.Tensor,
                   h0: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Training form of ``gru_head``: (lin(GRUCell(h, h0)), GRUCell(h, h0)) as
    one autograd Function over gfd_gru_head / gfd_gru_head_bwd / gfd_atb
    (tgn.py:108-111 under loss.backward(), train.py:142)."""
    if gru.hidden_size != C or gru.input_size != C or not gru.bias:
        raise NotImplementedError("gfd tgn_head_train: GRUCell(64, 64) with biases")
    x = _aligned_rows(h if h.dtype == torch.float32 else h.float())
    if h0 is not None:
        h0 = _aligned_rows(h0.float() if h0.dtype != torch.float32 else h0)
    b_o = lin.bias
    return _GRUHeadTrain.apply(x, h0, gru.weight_ih.contiguous(), gru.bias_ih,
                               gru.weight_hh.contiguous(), gru.bias_hh, lin.weight.contiguous(),
                               b_o)


class _BNReluDropout(torch.autograd.Function):
    """out = res + dropout(relu(bn_train(y))); see include/gfd.h gfd_bn_relu_fwd."""

    @staticmethod
    def forward(ctx, y, res, gamma, beta, bn, relu, p, seed):
        dev = y.device
        N = y.size(0)
        lib = _lib.load()
        ws = _ws(lib.gfd_bn_workspace_size(), dev)
        out = torch.empty_like(y)
        mean = torch.empty(C, dtype=torch.float32, device=dev)
        invstd = torch.empty_like(mean)
        momentum = bn.momentum
        if bn.track_running_stats and bn.num_batches_tracked is not None:
            bn.num_batches_tracked.add_(1)
            if momentum is None:  # cumulative moving average (torch BatchNorm semantics)
                momentum = 1.0 / float(bn.num_batches_tracked.item())
        rm = bn.running_mean if bn.track_running_stats else None
        rv = bn.running_var if bn.track_running_stats else None
        _lib.call("gfd_bn_relu_fwd", y.data_ptr(), _lib.ptr(res), N, C, _lib.ptr(gamma),
                  _lib.ptr(beta), float(bn.eps), float(momentum or 0.0), _lib.ptr(rm),
                  _lib.ptr(rv), 1 if relu else 0, float(p), seed, out.data_ptr(),
                  mean.data_ptr(), invstd.data_ptr(), ws.data_ptr(), ws.numel(),
                  _lib.stream_handle(dev))
        if rm is not None:                      # written by the call: what eval_weights goes by
            torch.autograd.graph.increment_version([rm, rv])
        ctx.save_for_backward(y, gamma, beta, mean, invstd)
        ctx.relu, ctx.p, ctx.seed, ctx.has_res = relu, p, seed, res is not None
        return out

    @staticmethod
    def backward(ctx, gout):
        y, gamma, beta, mean, invstd = ctx.saved_tensors
        gout = gout.contiguous()
        dev = y.device
        lib = _lib.load()
        ws = _ws(lib.gfd_bn_workspace_size(), dev)
        gy = torch.empty_like(y)
        gg = torch.empty(C, dtype=torch.float32, device=dev)
        gb = torch.empty_like(gg)
        _lib.call("gfd_bn_relu_bwd", y.data_ptr(), gout.data_ptr(), y.size(0), C,
                  gamma.data_ptr(), beta.data_ptr(), mean.data_ptr(), invstd.data_ptr(),
                  1 if ctx.relu else 0, float(ctx.p), ctx.seed, gy.data_ptr(), gg.data_ptr(),
                  gb.data_ptr(), ws.data_ptr(), ws.numel(), _lib.stream_handle(dev))
        return (gy, gout if ctx.has_res else None, gg, gb, None, None, None, None)


def train_supported(bn, y: torch.Tensor) -> bool:
    """Whether ``train_body`` takes this layer: an affine training-mode
    BatchNorm1d(64) over fp32 [N, 64] rows on the GPU."""
    return (bn is not None and bn.training and bn.affine and y.is_cuda
            and y.dtype == torch.float32 and y.dim() == 2 and y.size(1) == C and y.size(0) > 1
            and bn.weight.dtype == torch.float32)


def train_body(y: torch.Tensor, bn: torch.nn.BatchNorm1d, h: Optional[torch.Tensor],
               relu: bool = True, p: float = 0.0) -> torch.Tensor:
    """(h +) dropout(relu(bn(y)), p) in training mode (gat.py:82-91).  The
    dropout mask is drawn from a seed taken from torch's CPU generator, so
    ``torch.manual_seed`` makes it reproducible (it is not torch's own mask)."""
    y = y.contiguous()
    res = None
    if h is not None:
        res = h if (h.dtype == torch.float32 and h.is_contiguous()) else h.float().contiguous()
    seed = int(torch.randint(0, 2 ** 62, (1,)).item()) if p > 0 else 0
    return _BNReluDropout.apply(y, res, bn.weight, bn.bias, bn, relu, p, seed)


# ---------------------------------------------------------------------------
# row-wise training operators
# ---------------------------------------------------------------------------

_ROW_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16,
               torch.float16: _lib.DTYPE_F16}
ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3}


def _check_rows(what: str, name: str, t: torch.Tensor) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"gfd {what}: {name} must be on a HIP device (got {t.device})")
    if t.dtype not in _ROW_DTYPES:
        raise TypeError(f"gfd {what}: {name} must be float32, bfloat16 or float16 (got {t.dtype})")


def _norm_shape(x, ptr, groups) -> tuple:
    """The arguments of the group norm's C calls that say how x lies."""
    ragged = ptr is not None
    segments, length = (ptr.numel() - 1, x.size(0)) if ragged else (x.size(0), x.size(1))
    return (_ROW_DTYPES[x.dtype], segments, length, _lib.ptr(ptr), x.size(-1), groups, x.stride(-2),
            0 if ragged else x.stride(0))


def _group_norm_fwd(x, weight, bias, ptr, groups, eps, act, keep):
    """(y, statistics or None, _norm_shape's, GFD_DTYPE_* of the affine)."""
    dev, ragged = x.device, ptr is not None
    shape = _norm_shape(x, ptr, groups)
    _, segments, length, _, C, _, _, _ = shape
    y = torch.empty(x.shape, dtype=x.dtype, device=dev)
    # a row of its own keeps no statistics: the backward finds them again
    stats = (torch.empty((segments, groups, 2), dtype=torch.float64, device=dev)
             if keep and (ragged or length != 1) else None)
    w_dtype = _ROW_DTYPES[weight.dtype if weight is not None else
                          bias.dtype if bias is not None else x.dtype]
    nbytes = _lib.load().gfd_group_norm_workspace_size(segments, length, int(ragged), C, groups, 0)
    ws = _ws(nbytes, dev) if nbytes else None
    _lib.call_on(dev, "gfd_group_norm_fwd", x.data_ptr(), *shape, _lib.ptr(weight), _lib.ptr(bias),
                 w_dtype, eps, act, y.data_ptr(), _lib.ptr(stats), _lib.ptr(ws), nbytes,
                 _lib.stream_handle(dev))
    return y, stats, shape, w_dtype


class _GroupNorm(torch.autograd.Function):
    """act(group_norm(x)) over gfd_group_norm_fwd / _bwd; x [B, L, C] (dense) or
    [N, C] with ptr (ragged).  x and, but for single rows, the fp64 statistics are
    kept."""

    @staticmethod
    def forward(ctx, x, weight, bias, ptr, groups, eps, act):
        y, stats, ctx.shape, ctx.w_dtype = _group_norm_fwd(x, weight, bias, ptr, groups, eps, act, True)
        ctx.save_for_backward(x, weight, bias, ptr, stats)
        ctx.act, ctx.eps, ctx.strides = act, eps, x.stride()
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, weight, bias, ptr, stats = ctx.saved_tensors
        shape = ctx.shape
        _, segments, length, at, C, groups, _, _ = shape
        if x.stride() != ctx.strides or at != _lib.ptr(ptr) or _gaps(weight, bias, ptr, stats):
            # saved-tensor hooks brought them back elsewhere, or in other strides
            x = _unit_rows(x)
            weight, bias, ptr, stats = map(_packed, (weight, bias, ptr, stats))
            shape = _norm_shape(x, ptr, groups)
        dev = x.device
        grad = grad.contiguous()
        gx = torch.empty(x.shape, dtype=x.dtype, device=dev)
        gw = torch.empty_like(weight) if weight is not None and ctx.needs_input_grad[1] else None
        gb = torch.empty_like(bias) if bias is not None and ctx.needs_input_grad[2] else None
        nbytes = _lib.load().gfd_group_norm_workspace_size(segments, length, int(ptr is not None), C,
                                                           groups, 1)
        ws = _ws(nbytes, dev)
        _lib.call_on(dev, "gfd_group_norm_bwd", x.data_ptr(), *shape, _lib.ptr(weight),
                     _lib.ptr(bias), ctx.w_dtype, ctx.eps, ctx.act, _lib.ptr(stats), grad.data_ptr(),
                     gx.data_ptr(), _lib.ptr(gw), _lib.ptr(gb), ws.data_ptr(), ws.numel(),
                     _lib.stream_handle(dev))
        return gx, gw, gb, None, None, None, None


def _gaps(*tensors) -> bool:
    """Whether one of them (None: none) is not contiguous."""
    for t in tensors:
        if t is not None and not t.is_contiguous():
            return True
    return False


def _packed(t):
    """``t`` contiguous (None for None)."""
    return t if t is None else t.contiguous()


def _unit_rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` whose last dimension has no gaps."""
    return t if t.size(-1) <= 1 or t.stride(-1) == 1 else t.contiguous()


def _needs_grad(*tensors) -> bool:
    """Whether autograd has to see a call: for a gradient, or, while a forward-mode level is open,
    for a tangent, which the functions refuse."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        return True
    return forward_ad._current_level >= 0 and any(
        t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def group_norm(x: torch.Tensor, num_groups: int, weight: Optional[torch.Tensor] = None,
               bias: Optional[torch.Tensor] = None, eps: float = 1e-5, act: str = "none",
               ptr: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``act(group_norm(x) * weight + bias)``, channels last, differentiable.

    x [N, C]: every row has its own statistics over the channels of a group;
    x [B, ..., C]: over all positions of a sample and the channels of a group;
    x [N, C] with ``ptr`` (int64 [segments + 1] on the device, non-decreasing, as
    a ragged batch of graphs has): over the rows ptr[s] .. ptr[s + 1] of a
    segment, which may be empty.  Rows outside of every segment get 0 and no
    gradient.  x in float32, bfloat16 or float16, C <= 2048; weight / bias [C]
    in float32 or x's type; ``act`` none, relu, silu or gelu (erf).  The output
    is contiguous."""
    _check_rows("group_norm", "x", x)
    if act not in ACTIVATIONS:
        raise ValueError(f"gfd group_norm: act must be one of {sorted(ACTIVATIONS)} (got {act!r})")
    if x.dim() < 2 or (ptr is not None and x.dim() != 2):
        raise ValueError(f"gfd group_norm: x must be [N, C] or [B, ..., C], with ptr [N, C] (got "
                         f"{tuple(x.shape)})")
    C = x.size(-1)
    if not 1 <= C <= 2048:
        raise NotImplementedError(f"gfd group_norm: 1 to 2048 channels (got {C})")
    if num_groups < 1 or C % num_groups:
        raise ValueError(f"gfd group_norm: {C} channels are not a multiple of {num_groups} groups")
    if not eps >= 0:
        raise ValueError(f"gfd group_norm: eps must be >= 0 (got {eps})")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if t.device != x.device:
            raise RuntimeError(f"gfd group_norm: {name} is on {t.device}, expected {x.device}")
        if t.shape != (C,):
            raise ValueError(f"gfd group_norm: {name} must be [{C}] (got {tuple(t.shape)})")
        if t.dtype not in (torch.float32, x.dtype) or (weight is not None and t.dtype != weight.dtype):
            raise TypeError(f"gfd group_norm: weight and bias must both be float32 or {x.dtype} "
                            f"(got {name} {t.dtype})")
    if ptr is not None:
        if ptr.device != x.device or ptr.dtype != torch.int64 or ptr.dim() != 1 or ptr.numel() < 1:
            raise ValueError("gfd group_norm: ptr must be int64 [segments + 1] on x's device")
        ptr = ptr.contiguous()
    shape = x.shape
    if ptr is None:
        x = x.unsqueeze(1) if x.dim() == 2 else x.flatten(1, -2)
    if C > 1 and x.stride(-1) != 1:
        x = x.contiguous()
    weight = weight.contiguous() if weight is not None else None
    bias = bias.contiguous() if bias is not None else None
    args = (x, weight, bias, ptr, int(num_groups), float(eps), ACTIVATIONS[act])
    y = _GroupNorm.apply(*args) if _needs_grad(x, weight, bias) else _group_norm_fwd(*args, False)[0]
    return y if y.shape == shape else y.view(shape)


class ClassLogProbs(NamedTuple):
    """What ``class_log_probs`` returns; all float32 but the classes (int64)."""
    log_prob: Optional[torch.Tensor]     # [...] of the given classes; None without a target
    entropy: torch.Tensor                # [...] natural log
    top_log_probs: torch.Tensor          # [..., top]
    top_classes: torch.Tensor            # [..., top]


def _class_log_probs_fwd(logits, target, top, ignore_index, keep=False):
    """(logp, entropy, top_logp, top_class, statistics or None, the leading arguments of the C
    calls)."""
    dev = logits.device
    rows, classes = logits.shape
    f32 = dict(dtype=torch.float32, device=dev)
    logp = torch.empty(rows, **f32) if target is not None else None
    entropy = torch.empty(rows, **f32)
    top_logp = torch.empty((rows, top), **f32)
    top_class = torch.empty((rows, top), dtype=torch.int64, device=dev)
    nbytes = _lib.load().gfd_class_logp_workspace_size(rows, classes, top)
    # statistics that nobody keeps lie behind the workspace: an allocation less
    stats = torch.empty((rows, 2), **f32) if keep else None
    behind = -(-nbytes // 16) * 16
    ws = _ws(nbytes if keep else behind + 8 * rows, dev) if nbytes or not keep else None
    shape = (_ROW_DTYPES[logits.dtype], rows, classes, logits.stride(0))
    _lib.call_on(dev, "gfd_class_logp_fwd", logits.data_ptr(), *shape, _lib.ptr(target),
                 ignore_index, top, _lib.ptr(logp), entropy.data_ptr(), top_logp.data_ptr(),
                 top_class.data_ptr(), stats.data_ptr() if keep else ws.data_ptr() + behind,
                 _lib.ptr(ws), nbytes,
                 _lib.stream_handle(dev))
    return logp, entropy, top_logp, top_class, stats, shape


class _ClassLogProbs(torch.autograd.Function):
    """Over gfd_class_logp_fwd / _bwd: the logits, two statistics and the entropy
    of a row are kept."""

    @staticmethod
    def forward(ctx, logits, target, top, ignore_index):
        logp, entropy, top_logp, top_class, stats, ctx.shape = _class_log_probs_fwd(
            logits, target, top, ignore_index, True)
        ctx.save_for_backward(logits, target, entropy, top_class, stats)
        ctx.top, ctx.ignore_index, ctx.strides = top, ignore_index, logits.stride()
        ctx.mark_non_differentiable(top_class)
        ctx.set_materialize_grads(False)
        return logp, entropy, top_logp, top_class

    @staticmethod
    @once_differentiable
    def backward(ctx, g_logp, g_entropy, g_top, _):
        logits, target, entropy, top_class, stats = ctx.saved_tensors
        shape = ctx.shape
        if logits.stride() != ctx.strides or _gaps(target, entropy, top_class, stats):
            # saved-tensor hooks brought them back in other strides
            logits = _unit_rows(logits)
            target, entropy, top_class, stats = map(_packed, (target, entropy, top_class, stats))
            shape = shape[:3] + (logits.stride(0),)
        dev = logits.device
        g_logp, g_entropy, g_top = map(_packed, (g_logp, g_entropy, g_top))
        grad = torch.empty(logits.shape, dtype=logits.dtype, device=dev)
        _lib.call_on(dev, "gfd_class_logp_bwd", logits.data_ptr(), *shape, _lib.ptr(target),
                     ctx.ignore_index, ctx.top, top_class.data_ptr(), stats.data_ptr(),
                     entropy.data_ptr(), _lib.ptr(g_logp), _lib.ptr(g_entropy), _lib.ptr(g_top),
                     grad.data_ptr(), _lib.stream_handle(dev))
        return grad, None, None, None


def class_log_probs(logits: torch.Tensor, target: Optional[torch.Tensor] = None, top: int = 0,
                    ignore_index: int = -1) -> ClassLogProbs:
    """Log probabilities of the given classes, the entropy and the ``top`` most
    likely classes with their log probabilities, for logits [..., classes] in
    float32, bfloat16 or float16 and target int64 [...]; differentiable in the
    log probabilities and the entropy.

    A target of ``ignore_index`` (the reference's unknown label, -1) has log
    probability 0 and no gradient; any other one outside of the classes gives NaN.
    A masked class is a logit of -inf; a row of nothing else has log probability
    -inf, entropy 0 and no gradient.  Equal logits are listed by the lower class.
    0 <= top <= min(64, classes)."""
    _check_rows("class_log_probs", "logits", logits)
    if logits.dim() < 1 or logits.size(-1) < 1:
        raise ValueError(f"gfd class_log_probs: logits must be [..., classes] (got {tuple(logits.shape)})")
    classes, lead = logits.size(-1), logits.shape[:-1]
    if not 0 <= top <= min(64, classes):
        raise ValueError(f"gfd class_log_probs: top must be in [0, {min(64, classes)}] (got {top})")
    if target is not None:
        if target.device != logits.device:
            raise RuntimeError(f"gfd class_log_probs: target is on {target.device}, expected "
                               f"{logits.device}")
        if target.dtype != torch.int64:
            raise TypeError(f"gfd class_log_probs: target must be int64 (got {target.dtype})")
        if target.shape != lead:
            raise ValueError(f"gfd class_log_probs: target must be {tuple(lead)} (got "
                             f"{tuple(target.shape)})")
        target = target.reshape(-1).contiguous()
    x = logits if logits.dim() == 2 else logits.reshape(-1, classes)
    x = _unit_rows(x)
    args = (x, target, int(top), int(ignore_index))
    logp, entropy, top_logp, top_class = (_ClassLogProbs.apply(*args) if _needs_grad(x) else
                                          _class_log_probs_fwd(*args)[:4])
    if logits.dim() == 2:
        return ClassLogProbs(logp, entropy, top_logp, top_class)
    return ClassLogProbs(logp.view(lead) if logp is not None else None, entropy.view(lead),
                         top_logp.view(*lead, top), top_class.view(*lead, top))
