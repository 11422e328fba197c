"""Top alternatives and distillation through the fused vocabulary projection: what ``topk_logprobs_from_logits`` and
``topk_distillation_from_logits`` (``verl_amd/utils/torch_functional.py``) do for materialised logits, from the hidden states and
the weight of the head.

A teacher's pass is ``linear_topk_logprobs``; its two last results are what a student's ``linear_topk_distillation`` takes.  Both
run on the tile engine of ``linear_cross_entropy``, with its shapes and checks.
"""
from __future__ import annotations

import torch

from ... import _cabi
from ..torch_functional import divergence_code
from .linear_cross_entropy import _check_inputs, _new_logits_cache, active_token_index, keeps_logits

TOPK_MAX = 256   # VAMD_TOPK_MAX
FEW_TOKENS = 128   # up to which the head's kernels are bound by reading the weight


def _check_temperature(temperature: float) -> None:
    assert isinstance(temperature, float), f"temperature must be a float, but got {type(temperature)}"
    assert 0.0 < 1.0 / temperature < float("inf") if temperature > 0.0 else False, (
        f"temperature must be positive, but got {temperature}")


@torch.no_grad()
def linear_topk_logprobs(hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor | None, k: int,
                         temperature: float = 1.0):
    """``(logprobs, entropy, topk_logprobs, topk_indices)`` of ``softmax(hidden @ weight.T / temperature)``, without gradients.

    hidden ``(..., hidden_size)`` bf16, weight ``(vocab_size, hidden_size)`` bf16, labels ``(...)`` or ``None`` (then ``logprobs`` is
    ``None``).  fp32 results in the leading dimensions of ``hidden``, the last two (indices int64) with one dimension of ``k`` more:
    the ``k`` largest logits, largest first, the lowest index first among equals, ``1 <= k <= min(256, vocab_size)``.  The logits of
    a few thousand tokens at a time are held in a workspace."""
    _check_temperature(temperature)
    assert isinstance(k, int) and 1 <= k <= min(TOPK_MAX, weight.shape[0]), (
        f"k must be 1 to {TOPK_MAX} and at most the vocabulary, got {k} for {weight.shape[0]}")
    lead = hidden.shape[:-1]
    hidden = hidden.reshape(-1, hidden.shape[-1])
    n, h = hidden.shape
    dev = hidden.device
    if labels is None:
        given = torch.zeros(n, dtype=torch.int64, device=dev)
    else:
        assert labels.shape == lead, f"labels {tuple(labels.shape)} do not match hidden states {(*lead, h)}"
        given = labels.reshape(-1)
    _check_inputs(hidden, weight, given)
    if given.dtype != torch.int64:
        given = given.to(torch.int64)
    v = weight.shape[0]
    f32 = lambda *shape: torch.empty(shape, dtype=torch.float32, device=dev)
    logprobs, entropy, top = f32(n), f32(n), f32(n, k)
    index = torch.empty((n, k), dtype=torch.int64, device=dev)
    if n > 0:
        L = _cabi.lib()
        with _cabi.device_guard(dev):   # the query as well: it counts the current device's compute units
            ws = _cabi.workspace(L.vamd_lce_topk_workspace_bytes(n, h, v, k, 0), dev)
            _cabi.check(L.vamd_lce_topk(hidden.data_ptr(), weight.data_ptr(), given.data_ptr(), n, h, v, k, 1.0 / temperature,
                                        logprobs.data_ptr(), entropy.data_ptr(), top.data_ptr(), index.data_ptr(), 0,
                                        ws.data_ptr(), ws.numel(), _cabi.stream_ptr(dev)))
    return (None if labels is None else logprobs.view(lead), entropy.view(lead), top.view(*lead, k), index.view(*lead, k))


def _backward(d_loss, hidden, weight, no_labels, index, lse, slope_sum, slope, prob, temperature, need_dh, need_dw, cache,
              planned=None, rows=None):
    """Both gradients over the tokens given; ``rows`` and ``planned`` as in ``efficient_entropy_backward``."""
    n, h = hidden.shape
    v, k = weight.shape[0], index.shape[1]
    dev = hidden.device
    planned = n if planned is None else planned
    d_hidden = torch.empty_like(hidden) if need_dh else None
    d_weight = torch.empty_like(weight) if need_dw else None
    d_slope = d_loss * slope_sum
    L = _cabi.lib()
    with _cabi.device_guard(dev):
        ws = _cabi.workspace(L.vamd_lce_backward_subset_workspace_bytes(n, planned, h, v, 0), dev)
        _cabi.check(L.vamd_lce_divergence_backward(
            hidden.data_ptr(), weight.data_ptr(), no_labels.data_ptr(), n, planned, h, v, index.data_ptr(), k,
            1.0 / temperature, lse.data_ptr(), slope_sum.data_ptr(), slope.data_ptr(), prob.data_ptr(), d_loss.data_ptr(),
            d_slope.data_ptr(), _cabi.ptr(cache), _cabi.ptr(rows), _cabi.ptr(d_hidden), _cabi.ptr(d_weight),
            _cabi.DW_STORE if need_dw else _cabi.DW_NONE, None, 0, ws.data_ptr(), ws.numel(), _cabi.stream_ptr(dev)))
    return d_hidden, d_weight


class LinearTopkDistillation(torch.autograd.Function):
    """``linear_topk_distillation``'s node; ``grad_mode`` as in ``LinearCrossEntropy``."""

    @staticmethod
    def forward(ctx, hidden, weight, teacher_logprobs, teacher_indices, code: int, beta: float, temperature: float,
                grad_mode: bool = True):
        ctx.set_materialize_grads(False)
        lead = hidden.shape[:-1]
        shape = hidden.shape
        hidden = hidden.reshape(-1, shape[-1])
        n, v, dev = hidden.shape[0], weight.shape[0], hidden.device
        k = teacher_indices.shape[-1]
        t = teacher_logprobs.detach().reshape(-1, k).to(device=dev, dtype=torch.float32).contiguous()
        index = teacher_indices.reshape(-1, k).to(device=dev, dtype=torch.int64).contiguous()
        follows = grad_mode and (ctx.needs_input_grad[0] or ctx.needs_input_grad[1])
        cache = _new_logits_cache(n, v, dev) if follows and keeps_logits(n, v, dev) else None
        no_labels = torch.full((n,), -1, dtype=torch.int64, device=dev)
        _check_inputs(hidden, weight, no_labels)
        lse, rest, scratch, loss = (torch.empty(s, dtype=torch.float32, device=dev) for s in (n, n, 3 * n, n))
        slope_sum, slope, prob = (torch.empty(s, dtype=torch.float32, device=dev) if follows else None
                                  for s in ((n,), (n, k), (n, k)))
        L, h = _cabi.lib(), hidden.shape[1]
        with _cabi.device_guard(dev):   # the query as well: it counts the current device's compute units
            ws = _cabi.workspace(L.vamd_lce_forward_workspace_bytes(n, h, v), dev)
            _cabi.check(L.vamd_lce_divergence_forward(
                hidden.data_ptr(), weight.data_ptr(), no_labels.data_ptr(), n, h, v, 1.0 / temperature, scratch.data_ptr(),
                lse.data_ptr(), rest.data_ptr(), _cabi.ptr(cache), ws.data_ptr(), ws.numel(), _cabi.stream_ptr(dev)))
            _cabi.check(L.vamd_lce_divergence(
                hidden.data_ptr(), weight.data_ptr(), _cabi.ptr(cache), n, h, v, t.data_ptr(), index.data_ptr(), k,
                code, beta, 1.0 / temperature, lse.data_ptr(), rest.data_ptr(), loss.data_ptr(), _cabi.ptr(slope_sum), _cabi.ptr(slope),
                _cabi.ptr(prob), _cabi.stream_ptr(dev)))
        ctx.save_for_backward(hidden, weight, no_labels, index, lse, slope_sum, slope, prob, cache)
        ctx.hidden_shape = shape
        ctx.temperature = temperature
        return loss.view(lead)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_loss):
        hidden, weight, no_labels, index, lse, slope_sum, slope, prob, cache = ctx.saved_tensors
        need_dh, need_dw = ctx.needs_input_grad[:2]
        if d_loss is None or not (need_dh or need_dw):
            return (None,) * 8
        g = d_loss.reshape(-1).to(torch.float32).contiguous()
        # tokens that the loss masked out are left out of the kernels, as in linear_cross_entropy; not of few, over which they wait
        # for the weight, however many there are (93 x 896 x 151936, an eighth of them masked out: 360 us with and 247 without)
        idx = active_token_index(g, None, hidden.shape[0], weight.shape) if hidden.shape[0] > FEW_TOKENS else None
        if idx is None:
            d_hidden, d_weight = _backward(g, hidden, weight, no_labels, index, lse, slope_sum, slope, prob, ctx.temperature,
                                           need_dh, need_dw, cache)
        else:
            d_hidden = torch.zeros_like(hidden) if need_dh else None
            d_weight = None
            if idx.numel() == 0:
                d_weight = torch.zeros_like(weight) if need_dw else None
            else:
                take = lambda x: x.index_select(0, idx)
                dh, d_weight = _backward(take(g), take(hidden), weight, no_labels[:idx.numel()], take(index), take(lse), take(slope_sum), take(slope),
                                         take(prob), ctx.temperature, need_dh, need_dw, cache, hidden.shape[0],
                                         None if cache is None else idx)
                if need_dh:
                    d_hidden.index_copy_(0, idx, dh)
        return (None if d_hidden is None else d_hidden.view(ctx.hidden_shape), d_weight, None, None, None, None, None, None)


def linear_topk_distillation(hidden: torch.Tensor, weight: torch.Tensor, teacher_logprobs: torch.Tensor,
                             teacher_indices: torch.Tensor, divergence: str = "forward_kl", beta: float = 0.5,
                             temperature: float = 1.0) -> torch.Tensor:
    """Divergence of ``softmax(hidden @ weight.T / temperature)`` from a teacher's most likely tokens, per token: fp32 in the leading
    dimensions of ``hidden``, differentiable once in ``hidden`` and ``weight`` (bf16).  The divergences, and what a padding entry
    is, are ``topk_distillation_from_logits``'.

    A forward pass that a backward pass will follow keeps its logits as ``linear_cross_entropy`` does, and the backward pass
    leaves out the tokens whose upstream gradient is zero, as that does."""
    code = divergence_code(divergence, beta)
    _check_temperature(temperature)
    assert teacher_logprobs.shape == teacher_indices.shape and teacher_indices.shape[:-1] == hidden.shape[:-1], (
        f"the teacher's log-probs {tuple(teacher_logprobs.shape)} and indices {tuple(teacher_indices.shape)} must have the shape "
        f"of the tokens {tuple(hidden.shape[:-1])} and one dimension more")
    assert 1 <= teacher_indices.shape[-1] <= TOPK_MAX, (
        f"a teacher's tokens must be 1 to {TOPK_MAX}, got {teacher_indices.shape[-1]}")
    assert teacher_logprobs.is_floating_point(), "the teacher's log-probs must be of a floating type"
    assert teacher_indices.dtype in (torch.int64, torch.int32), f"the teacher's indices must be int64 or int32, got {teacher_indices.dtype}"
    assert hidden.is_cuda and weight.is_cuda and hidden.numel() > 0
    if torch.is_grad_enabled():
        for x in (hidden, weight):
            _cabi.ops().refuse_capture_beside_eager_graph("linear_topk_distillation", x)
    return LinearTopkDistillation.apply(hidden, weight, teacher_logprobs, teacher_indices, code, float(beta), temperature,
                                        torch.is_grad_enabled())
