"""Top alternatives and distillation through the vocabulary projection: GPU kernels against the oracle (oracle/topk.py) in 64 bits.

Tolerances (u = 2^-24): a logit is a sum of H products whose roundings add up to at most H u sum |h w|, half of it per addition;
together with the softmax's sum, (V / 256 + 64) u as in tests/test_gpu_topk.py, that is the error E of a log-probability.  The
gradients go through d_logits in bf16 (half a step, 2^-8 of each) and are rounded to bf16 once more.  Where indices are compared the
inputs are multiples of 1/8 and 1/512, so that every sum is exact in fp32.
"""
import math

import pytest
import torch

import oracle as O

U = 2.0 ** -24
KINDS = ["forward_kl", "reverse_kl", "jsd"]
INF, NAN = math.inf, math.nan
gpu = pytest.mark.gpu


def _head(n, h, v, seed):
    g = torch.Generator().manual_seed(seed)
    hidden = (torch.randn(n, h, generator=g) * 8).round().clamp(-31, 31) / 8
    weight = (torch.randn(v, h, generator=g) * 512 * 1.5 / math.sqrt(h)).round().clamp(-120, 120) / 512
    return hidden.bfloat16(), weight.bfloat16()


def _error(hidden, weight, temperature):
    h, v = hidden.shape[-1], weight.shape[0]
    size = (hidden.double().abs() @ weight.double().abs().t()).amax().item() / temperature
    return h * U * size + (v / 256 + 64) * U + 40 * U * (size ** 0.5 + 20)


def _close(got, want, bound, what):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, what
    err = (got - want).abs()
    bound = torch.as_tensor(bound, dtype=torch.float64).expand_as(want)
    assert bool((err <= bound).all()), f"{what}: off by {err.max().item():.3e}, {(err / bound).max().item():.2f} of the bound"


@gpu
@pytest.mark.parametrize("n,h,v,k,temperature", [
    (1, 128, 300, 5, 1.0), (5, 256, 1001, 7, 0.7), (93, 128, 4099, 64, 1.0), (128, 384, 2049, 256, 1.3), (129, 256, 3002, 20, 1.0),
    (300, 128, 5003, 256, 1.0), (700, 640, 1007, 65, 0.7), (4, 128, 1, 1, 1.0), (200, 128, 30, 30, 1.0), (260, 128, 33003, 9, 1.0)])
def test_topk(dev, n, h, v, k, temperature):
    from verl_amd.utils.kernel.linear_topk import linear_topk_logprobs
    hidden, weight = _head(n, h, v, n + v)
    if v > 500:   # equal logits: rows of the weight that are the same
        weight[400] = weight[11]
        weight[v - 1] = weight[11]
        weight[256:260] = weight[2]
    labels = torch.randint(0, v, (n,), generator=torch.Generator().manual_seed(n))
    lp, ent, top, index = linear_topk_logprobs(hidden.to(dev), weight.to(dev), labels.to(dev), k, temperature)
    want_lp, want_ent, want_top, want_index = O.topk_logprobs(hidden.double() @ weight.double().t(), labels, k, temperature)
    e = _error(hidden, weight, temperature)
    assert torch.equal(index.cpu(), want_index)
    _close(lp, want_lp, e, "logprobs")
    _close(top, want_top, e, "top")
    _close(ent, want_ent, e * (2 + want_ent.abs()), "entropy")


@gpu
def test_topk_of_leading_dimensions_chunks_and_strides(dev):
    """Leading dimensions, no labels, int32 labels, no tokens; chunks of tokens give the same bits, whatever lies in the workspace."""
    from verl_amd import _cabi
    from verl_amd.utils.kernel.linear_topk import linear_topk_logprobs
    n, h, v, k = 650, 128, 3003, 12
    hidden, weight = (x.to(dev) for x in _head(n, h, v, 3))
    labels = torch.randint(0, v, (n,), device=dev)
    whole = linear_topk_logprobs(hidden, weight, labels, k)
    lead = linear_topk_logprobs(hidden.view(13, 50, h), weight, labels.int().view(13, 50), k)
    for a, b in zip(whole, lead):
        assert b.shape[:2] == (13, 50) and torch.equal(a, b.reshape(a.shape))
    none = linear_topk_logprobs(hidden.view(13, 50, h).transpose(0, 1), weight, None, k)
    assert none[0] is None and torch.equal(none[3], whole[3].view(13, 50, k).transpose(0, 1))
    empty = linear_topk_logprobs(hidden[:0], weight, labels[:0], k)
    assert empty[0].shape == (0,) and empty[3].shape == (0, k)
    L = _cabi.lib()
    for chunk in (100, 256, 649, 650, 10**6):
        ws = torch.full((L.vamd_lce_topk_workspace_bytes(n, h, v, k, chunk),), 255, dtype=torch.uint8, device=dev)
        out = [torch.empty_like(x) for x in whole]
        _cabi.check(L.vamd_lce_topk(hidden.data_ptr(), weight.data_ptr(), labels.data_ptr(), n, h, v, k, 1.0,
                                    *(x.data_ptr() for x in out), chunk, ws.data_ptr(), ws.numel(), _cabi.stream_ptr(dev)))
        assert torch.equal(out[3], whole[3])
        for a, b in zip(out[:3], whole[:3]):
            assert (a - b).abs().max().item() <= 2 * _error(hidden.cpu(), weight.cpu(), 1.0)


def _teacher(hidden, weight, k, temperature, seed):
    z = hidden.float() @ weight.float().t()
    z = (z + torch.randn(z.shape, generator=torch.Generator().manual_seed(seed))) / temperature
    return z.log_softmax(-1).topk(k, -1)


def _distil(dev, hidden, weight, t, index, kind, beta, temperature, up, need=(True, True)):
    from verl_amd.utils.kernel.linear_topk import linear_topk_distillation
    hd, wd = hidden.to(dev).requires_grad_(need[0]), weight.to(dev).requires_grad_(need[1])
    loss = linear_topk_distillation(hd, wd, t.to(dev), index.to(dev), kind, beta, temperature)
    with torch.no_grad():
        again = linear_topk_distillation(hd, wd, t.to(dev), index.to(dev), kind, beta, temperature)
    inputs = [x for x, wanted in zip((hd, wd), need) if wanted]
    grads = list(torch.autograd.grad(loss, inputs, up.to(dev)))
    return loss, again, *(grads.pop(0) if wanted else None for wanted in need)


def _check(dev, hidden, weight, t, index, kind, beta=0.3, temperature=1.0, up=None, need=(True, True)):
    n, v = hidden.shape[0], weight.shape[0]
    if up is None:
        up = torch.randn(n, generator=torch.Generator().manual_seed(1))
    loss, again, dh, dw = _distil(dev, hidden, weight, t, index, kind, beta, temperature, up, need)
    z = (hidden.double() @ weight.double().t()).requires_grad_()
    want = O.topk_distillation(z, t.double(), index.long(), kind, beta, temperature)
    d, = torch.autograd.grad(want, z, up.double())
    e = _error(hidden, weight, temperature)
    lq = torch.log_softmax(z.detach() / temperature, -1)
    ok = (index >= 0) & (index < v) & (t != -INF)
    at = torch.where(ok, index, 0).long()
    lqk, tt = lq.gather(-1, at), torch.where(ok, t.double(), 0.0)
    mass = torch.where(ok, (tt.exp() + lqk.exp()) * (1 + (tt - lqk).abs()), 0.0)
    for got in (loss, again):   # with the logits kept and without
        _close(got, want.detach(), 2 * (e + 16 * U) * mass.sum(-1) + 2.0 ** -126, "loss")
    # d_logits: half a step of bf16 each, and the relative error e of the probabilities and slopes in it
    scale = up.double().abs()[:, None] / temperature
    inside = 2.0 ** -8 * 1.01 * d.abs() + 3 * e * (lq.exp() * mass.sum(-1, keepdim=True) * scale
                                                  + torch.zeros_like(d).scatter_add_(1, at, mass * scale))
    sums = 64 * U * max(1, n // 32, v // 32)   # of fp32 additions, relative to the sum of the terms' sizes
    for got, want_g, slack in ((dh, d @ weight.double(), (inside + sums * d.abs()) @ weight.double().abs()),
                               (dw, d.t() @ hidden.double(), (inside + sums * d.abs()).t() @ hidden.double().abs())):
        if got is not None:
            assert got.dtype == torch.bfloat16
            _close(got, want_g, slack + 2.0 ** -8 * 1.01 * (want_g.abs() + slack) + 2.0 ** -126, "gradient")
    return loss, dh, dw


@gpu
@pytest.mark.parametrize("cache", [None, "0"])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,h,v,k,temperature", [
    (1, 128, 304, 5, 1.0), (5, 256, 1001, 7, 0.7), (64, 128, 4096, 64, 1.0), (129, 256, 3000, 20, 1.0), (300, 128, 2051, 256, 1.3),
    (600, 384, 1504, 100, 1.0)])
def test_distillation(dev, monkeypatch, cache, kind, n, h, v, k, temperature):
    """With the logits kept (vocabularies that allow it) and without."""
    if cache is not None:
        monkeypatch.setenv("VAMD_LCE_LOGITS_CACHE_GB", cache)
    hidden, weight = _head(n, h, v, n + v)
    t, index = _teacher(hidden, weight, k, temperature, 2)
    _check(dev, hidden, weight, t, index, kind, 0.3, temperature)


@gpu
@pytest.mark.parametrize("cache", [None, "0"])
def test_distillation_of_padded_and_repeated_entries(dev, monkeypatch, cache):
    """Padding by index and by log-probability (its column keeps the other term of its gradient), rows of nothing else, indices that
    come several times, tokens without a gradient, several vocabulary chunks, 32-bit indices."""
    if cache is not None:
        monkeypatch.setenv("VAMD_LCE_LOGITS_CACHE_GB", cache)
    monkeypatch.setenv("VAMD_LCE_DZ_BUDGET_MB", "1")
    n, h, v, k = 200, 128, 3008, 70
    hidden, weight = _head(n, h, v, 5)
    t, index = _teacher(hidden, weight, k, 1.0, 7)
    index[0, 3:] = -1
    t[1, 5:] = -INF
    index[2] = -1
    t[3] = -INF
    index[4] = 2047
    t[4] = -6.0
    index[5, ::2] = 9
    t[5] = -5.0
    index[6, 0], index[6, 1] = v, 2**30
    up = torch.randn(n, generator=torch.Generator().manual_seed(3))
    for kind in KINDS:
        loss, dh, _ = _check(dev, hidden, weight, t, index.int(), kind, up=up)
        assert loss[2].item() == 0.0 and loss[3].item() == 0.0 and not dh[2:4].any()
    up[50:] = 0   # the loss masked most tokens out
    _, dh, _ = _check(dev, hidden, weight, t, index, "forward_kl", up=up)
    assert not dh[50:].any()
    _, dh, dw = _check(dev, hidden, weight, t, index, "jsd", up=torch.zeros(n))
    assert not dh.any() and not dw.any()


@gpu
def test_token_tiles_shared_out_in_bands_and_in_splits(dev):
    """24 token tiles x 200 vocabulary tiles run in bands, a sixth of the tokens in splits: the same alternatives and losses."""
    from verl_amd import _cabi
    from verl_amd.utils.kernel.linear_topk import linear_topk_distillation, linear_topk_logprobs
    n, h, v, k = 6144, 128, 51200, 12
    hidden, weight = (x.to(dev) for x in _head(n, h, v, 3))
    labels = torch.randint(0, v, (n,), device=dev)
    e = 2 * _error(hidden[:64].cpu(), weight[:2000].cpu(), 1.0) * 1.5   # (the largest of a part of the sums; the rest by a half)
    whole = linear_topk_logprobs(hidden, weight, labels, k)
    parts = [linear_topk_logprobs(hidden[i:i + 1024], weight, labels[i:i + 1024], k) for i in range(0, n, 1024)]
    L = _cabi.lib()
    # the partial states tell which way the tiles are shared out: 10 splits of 24 tiles, or (3 bands + 8 XCDs) x 32 columns
    assert L.vamd_lce_forward_workspace_bytes(n, h, v) == 11 * 32 * 256 * 20
    for i, name in enumerate(("logprobs", "entropy", "top", "index")):
        part = torch.cat([p[i] for p in parts])
        if name == "index":
            assert torch.equal(whole[i], part)
        else:
            assert (whole[i] - part).abs().max().item() <= e * 15, name
    hd = hidden.clone().requires_grad_()
    loss = linear_topk_distillation(hd, weight, whole[2] - 0.2, whole[3], "jsd")
    part = torch.cat([linear_topk_distillation(hidden[i:i + 1024], weight, whole[2][i:i + 1024] - 0.2, whole[3][i:i + 1024], "jsd")
                      for i in range(0, n, 1024)])
    assert (loss - part).abs().max().item() <= 4 * e
    assert torch.isfinite(torch.autograd.grad(loss.sum(), hd)[0]).all()


@gpu
@pytest.mark.parametrize("need", [(True, False), (False, True)])
def test_distillation_with_one_frozen_input(dev, need):
    hidden, weight = _head(300, 256, 2000, 8)
    t, index = _teacher(hidden, weight, 16, 1.0, 7)
    _, dh, dw = _check(dev, hidden, weight, t, index, "reverse_kl", need=need)
    assert (dh is None, dw is None) == (not need[0], not need[1])


@gpu
def test_gradients_against_differences(dev):
    """Central differences in 64 bits of the oracle along random directions, of which the fp32 oracle of the gradient is no part:
    the directional derivative of d_hidden and d_weight, whose entries are off by 2^-8 of their size twice over, half a step each."""
    n, h, v, k = 6, 128, 120, 10
    hidden, weight = _head(n, h, v, 4)
    t, index = _teacher(hidden, weight, k, 1.0, 3)
    up = torch.rand(n, generator=torch.Generator().manual_seed(2))
    f = lambda a, b: (O.topk_distillation(a @ b.t(), t.double(), index, "jsd", 0.4) * up).sum()
    g = torch.Generator().manual_seed(9)
    _, _, dh, dw = _distil(dev, hidden, weight, t, index, "jsd", 0.4, 1.0, up)
    for got, which in ((dh, 0), (dw, 1)):
        x = [hidden.double(), weight.double()]
        for _ in range(3):
            step = torch.randn(x[which].shape, generator=g, dtype=torch.float64) * 1e-4
            both = []
            for s in (1, -1):
                y = list(x)
                y[which] = y[which] + s * step
                both.append(f(*y).item())
            got64 = got.double().cpu()
            size = (got64.abs() * step.abs()).sum().item()
            assert abs((both[0] - both[1]) / 2 - (got64 * step).sum().item()) <= 3 * 2.0 ** -8 * size + 1e-12


@gpu
def test_a_teacher_and_a_student_with_leading_dimensions(dev):
    """The run as it is used: a teacher's alternatives, the student's loss on them, aggregated over a mask, both gradients; the same
    from materialised logits."""
    import verl_amd.utils.torch_functional as F
    from verl_amd.trainer.ppo.core_algos import agg_loss
    from verl_amd.utils.kernel.linear_topk import linear_topk_distillation, linear_topk_logprobs
    b, l, h, v, k, temperature = 3, 60, 256, 3000, 32, 0.8
    (th, tw), (sh, sw) = _head(b * l, h, v, 1), _head(b * l, h, v, 2)
    mask = (torch.arange(l)[None] < torch.tensor([60, 1, 0])[:, None]).float()
    labels = torch.randint(0, v, (b, l))
    _, _, top, index = linear_topk_logprobs(th.view(b, l, h).to(dev), tw.to(dev), labels.to(dev), k, temperature)
    hd, wd = sh.view(b, l, h).to(dev).requires_grad_(), sw.to(dev).requires_grad_()
    loss = linear_topk_distillation(hd, wd, top, index, temperature=temperature)
    assert loss.shape == (b, l)
    total = agg_loss(loss, mask.to(dev), "token-mean")
    dh, dw = torch.autograd.grad(total, (hd, wd))
    assert dh.shape == hd.shape and not dh[2].any()
    h64, w64 = sh.double().requires_grad_(), sw.double().requires_grad_()
    _, _, want_top, want_index = O.topk_logprobs(th.double() @ tw.double().t(), labels.view(-1), k, temperature)
    assert torch.equal(index.view(-1, k).cpu(), want_index)
    z = h64 @ w64.t()
    per_token = O.topk_distillation(z, want_top, want_index, temperature=temperature)
    want = (per_token * mask.view(-1)).sum() / mask.sum()
    d, = torch.autograd.grad(want, z, retain_graph=True)
    e = _error(sh, sw, temperature) + _error(th, tw, temperature)
    assert abs(total.item() - want.item()) <= 2 * e * (1 + abs(want.item()))
    inside = (2.0 ** -8 + 40 * e) * d.abs() + 2 * e / mask.sum()  * torch.softmax(z.detach() / temperature, -1) * (mask.view(-1, 1) > 0)
    for got, a64, slack in ((dh.view(-1, h), h64, inside @ sw.double().abs()), (dw, w64, inside.t() @ sh.double().abs())):
        want_g, = torch.autograd.grad(want, a64, retain_graph=True)
        _close(got, want_g, slack + 2.0 ** -8 * 1.01 * (want_g.abs() + slack) + 1e-9, "gradient")
    rows = F.topk_distillation_from_logits((sh.float() @ sw.float().t()).view(b, l, v).to(dev), top, index, temperature=temperature)
    assert (rows - loss).abs().max().item() <= 4 * e * 20


@gpu
def test_both_replay_from_a_graph(dev):
    """Captured twice (without the logits kept), replayed on two streams at once between eager work, on new inputs."""
    from verl_amd.utils.kernel.linear_topk import linear_topk_distillation, linear_topk_logprobs
    n, h, v, k = 300, 128, 2003, 16
    hidden, weight = (x.to(dev).requires_grad_() for x in _head(n, h, v, 0))
    labels = torch.randint(0, v, (n,), device=dev)

    def step():
        lp, ent, top, index = linear_topk_logprobs(hidden, weight, labels, k)
        loss = linear_topk_distillation(hidden, weight, top - 0.1, index, "reverse_kl")
        return [x.detach() for x in (lp, ent, top, index, loss, *torch.autograd.grad(loss.sum(), (hidden, weight)))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for i in range(4):
        fresh = _head(n, h, v, 20 + i)
        with torch.no_grad():
            hidden.copy_(fresh[0])
            weight.copy_(fresh[1])
        torch.cuda.synchronize()
        for (graph, _), s in zip(graphs, (torch.cuda.Stream(), torch.cuda.Stream())):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        want = step()
        for _, out in graphs:
            for a, b in zip(out, want):
                assert torch.equal(a, b)


@gpu
def test_refusals(dev):
    from verl_amd.utils.kernel.linear_topk import linear_topk_distillation, linear_topk_logprobs
    hidden, weight = (x.to(dev) for x in _head(4, 128, 300, 1))
    labels = torch.zeros(4, dtype=torch.int64, device=dev)
    for k in (0, 257, 301, 2.0):
        with pytest.raises(AssertionError, match="k must be"):
            linear_topk_logprobs(hidden, weight, labels, k)
    for temperature in (0.0, -1.0, INF, NAN, 1, 1e-320):
        with pytest.raises(AssertionError, match="temperature"):
            linear_topk_logprobs(hidden, weight, labels, 2, temperature)
    for bad in ((hidden.float(), weight, labels), (hidden, weight[:, :64], labels), (hidden, weight.t().contiguous().t(), labels),
                (hidden[:, :100].contiguous(), weight[:, :100].contiguous(), labels), (hidden, weight, labels[:3])):
        with pytest.raises(AssertionError):
            linear_topk_logprobs(*bad, 2)
    t, index = torch.zeros(4, 5, device=dev), torch.zeros(4, 5, dtype=torch.int64, device=dev)
    for a, b in ((t[:3], index[:3]), (t[:, :4], index), (t[0], index[0]), (t[:, :0], index[:, :0]), (t.long(), index),
                 (t, index.float())):
        with pytest.raises(AssertionError, match="teacher"):
            linear_topk_distillation(hidden, weight, a, b)
    with pytest.raises(AssertionError):
        linear_topk_distillation(hidden.float(), weight, t, index)
    with pytest.raises(AssertionError):
        linear_topk_distillation(hidden[:0], weight, t[:0], index[:0])
    x = hidden.clone().requires_grad_()
    d, = torch.autograd.grad(linear_topk_distillation(x, weight, t, index).sum() ** 2, x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        d.sum().backward()
    w = weight.clone().requires_grad_()
    alive = linear_topk_distillation(hidden, w, t, index)
    with pytest.raises(RuntimeError, match="eager graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.ones(1, device=dev)
            linear_topk_distillation(hidden, w, t, index)
    torch.cuda.synchronize()
    del alive


def test_refusals_on_the_host():
    from verl_amd import _cabi
    from verl_amd.utils.kernel.linear_topk import linear_topk_distillation, linear_topk_logprobs
    hidden, weight = _head(4, 128, 300, 1)
    t, index = torch.zeros(4, 5), torch.zeros(4, 5, dtype=torch.int64)
    with pytest.raises(AssertionError):
        linear_topk_logprobs(hidden, weight, None, 5)
    with pytest.raises(AssertionError):
        linear_topk_distillation(hidden, weight, t, index)
    with pytest.raises(ValueError, match="Invalid divergence"):
        linear_topk_distillation(hidden, weight, t, index, "kl")
    for beta in (0.0, 1.0, NAN):
        with pytest.raises(AssertionError, match="beta"):
            linear_topk_distillation(hidden, weight, t, index, "jsd", beta)
    lib, at = _cabi.lib(), 4096   # never read
    topk = lambda hidden=at, n=4, h=128, v=300, k=5, rcp=1.0, labels=at, top=at, ws=at, size=1 << 40: lib.vamd_lce_topk(
        hidden, at, labels, n, h, v, k, rcp, at, at, top, at, 0, ws, size, None)
    for bad in (dict(hidden=None), dict(n=0), dict(h=100), dict(v=0), dict(k=0), dict(k=257), dict(k=301), dict(rcp=0.0),
                dict(rcp=NAN), dict(rcp=INF), dict(labels=None), dict(top=None)):
        assert topk(**bad) == -1, bad
    need = lib.vamd_lce_topk_workspace_bytes(4, 128, 300, 5, 0)
    assert topk(size=need - 1) == -2 and topk(ws=None) == -2
    assert lib.vamd_lce_topk_workspace_bytes(100000, 3584, 152064, 64, 0) < 4 << 30   # a few thousand tokens at a time
    div = lambda hidden=at, cache=None, v=300, teacher=at, k=5, kind=0, beta=0.5, rcp=1.0, slope=at, prob=at: lib.vamd_lce_divergence(
        hidden, at, cache, 4, 128, v, teacher, at, k, kind, beta, rcp, at, at, at, at, slope, prob, None)
    for bad in (dict(hidden=None), dict(hidden=at + 8), dict(cache=at, v=300 + 1), dict(teacher=None), dict(k=0), dict(k=257),
                dict(kind=3), dict(kind=2, beta=0.0), dict(rcp=-1.0), dict(rcp=INF), dict(slope=None), dict(prob=None)):
        assert div(**bad) == -1, bad
    back = lambda index=at, k=5, d_loss=at, d_hidden=at, rcp=1.0, size=1 << 40: lib.vamd_lce_divergence_backward(
        at, at, at, 4, 4, 128, 300, index, k, rcp, at, at, at, at, d_loss, at, None, None, d_hidden, at, _cabi.DW_STORE, None, 0,
        at, size, None)
    for bad in (dict(index=None), dict(k=0), dict(k=257), dict(d_loss=None), dict(rcp=0.0)):
        assert back(**bad) == -1, bad
    assert back(size=16) == -2
