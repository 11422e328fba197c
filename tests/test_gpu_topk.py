"""Top alternatives and distillation from materialised logits: GPU kernels against the oracle (oracle/topk.py) in 64 bits.

Tolerances, from fp32 arithmetic (half a step is u = 2^-24).  A thread adds up at most V / 256 + 32 exponentials, then 16 partial
sums meet: the sum's relative error is at most (V / 256 + 64) u, which is the absolute error that it leaves in a
log-probability.  The exponents y = z log2(e) / T are off by 3 u |y - max y| (two rounded factors and a product) and an exponential by
2 u; maximum, logarithm and differences round values of the size of |log q| a few times: 8 u |log q|.  Whatever is weighted by a
probability (entropy, divergence, gradient) inherits these relative errors.  A gradient in a 16-bit type is rounded once more, by
half a step of that type.
"""
import math

import pytest
import torch

import oracle as O

INF, NAN = math.inf, math.nan
U = 2.0 ** -24
HALF_STEP = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}   # eps / 2
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
KINDS = ["forward_kl", "reverse_kl", "jsd"]
gpu = pytest.mark.gpu


def _sum_error(v):
    return (v / 256 + 64) * U


def _logits(shape, dtype, seed, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def _labels(n, v, seed):
    return torch.randint(0, v, (n,), generator=torch.Generator().manual_seed(seed + 1))


def _within(got, want, bound, what):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} and {tuple(want.shape)}"
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN elsewhere"
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), f"{what}: infinities elsewhere"
    err = (got - want).abs()[fine]
    bound = torch.as_tensor(bound, dtype=torch.float64).expand_as(want)[fine]
    assert bool((err <= bound).all()), f"{what}: off by {err.max().item():.3e}, {(err / bound).max().item():.2f} of the bound"


def _check_forward(F, dev, z, labels, k, temperature=1.0):
    v = z.shape[-1]
    lp, ent, top, index = F.topk_logprobs_from_logits(z.to(dev), labels.to(dev), k, temperature)
    want_lp, want_ent, want_top, want_index = O.topk_logprobs(z.double(), labels, k, temperature)
    assert lp.dtype == ent.dtype == top.dtype == torch.float32 and index.dtype == torch.int64
    assert torch.equal(index.cpu(), want_index), "other alternatives"
    e = _sum_error(v)
    reach = (z.double().nan_to_num(0, 0, 0).abs().amax(-1) / temperature).clamp(min=1.0)
    _within(lp, want_lp, e + 12 * U * (want_lp.abs().nan_to_num(0, 0, 0) + reach), "logprobs")
    _within(top, want_top, e + 12 * U * (want_top.abs().nan_to_num(0, 0, 0) + reach[..., None]), "top")
    _within(ent, want_ent, (2 * e + 24 * U) * (want_ent.abs().nan_to_num(0, 0, 0) + reach + 1), "entropy")


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,v,k,temperature", [
    (1, 1, 1, 1.0), (2, 7, 7, 1.0), (3, 300, 256, 0.7), (37, 1152, 64, 1.0), (5, 2000, 65, 3.0), (1, 151936, 20, 1.0),
    (3, 33001, 256, 1.0), (64, 128256, 5, 0.7), (520, 4099, 100, 1.0), (600, 32003, 8, 1.3), (270, 50257, 64, 1.0)])
def test_topk_forward(dev, dtype, n, v, k, temperature):
    import verl_amd.utils.torch_functional as F
    _check_forward(F, dev, _logits((n, v), dtype, n + v), _labels(n, v, n), k, temperature)


@gpu
@pytest.mark.parametrize("n", [2, 600])
@pytest.mark.parametrize("k", [1, 20, 64, 200])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_topk_of_equal_sorted_and_clustered_logits(dev, dtype, n, k):
    """Equal logits go by their column, whichever way the k-th largest is found; few rows are split, many are not."""
    import verl_amd.utils.torch_functional as F
    v = 40007
    ramp = torch.arange(v, dtype=torch.float32) / v * 8
    rows = [torch.full((v,), 1.5), torch.zeros(v), ramp, ramp.flip(0), (torch.arange(v) % 7).float(),
            -(torch.arange(v) % 300).float(), torch.where(torch.arange(v) % 8192 < 40, 9.0, 0.0) + ramp]
    rows[1][::3] = -0.0
    z = torch.stack([rows[i % len(rows)] for i in range(max(n, len(rows)))]).to(dtype)
    few = z[:len(rows)]
    labels = _labels(len(rows), v, k)
    if n < len(rows):
        _check_forward(F, dev, few, labels, k)
    else:   # the same rows over and over: compared with the first of each
        index = F.topk_logprobs_from_logits(z.to(dev), None, k)[3].cpu()
        want = O.topk_logprobs(few.double(), labels, k)[3]
        assert torch.equal(index, torch.stack([want[i % len(rows)] for i in range(n)]))


@gpu
@pytest.mark.parametrize("n", [1, 300, 600])
@pytest.mark.parametrize("k", [5, 100])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_topk_of_masked_logits(dev, dtype, n, k):
    """Logits of -inf, the type's lowest value, +inf and NaN; rows with fewer finite logits than alternatives, and none."""
    import verl_amd.utils.torch_functional as F
    v = 20011
    z = _logits((7, v), dtype, 5)
    z[0, 40:] = -INF
    z[1] = -INF
    z[1, [3, 9000, 20010]] = torch.tensor([2.0, 2.0, 1.0]).to(dtype)
    z[2, 50:] = torch.finfo(dtype).min
    z[3] = -INF
    z[4, 77] = NAN
    z[5] = NAN
    z[5, [11, 5000]] = -INF
    z[6, 5] = INF
    labels = torch.tensor([3, 9000, 50, 0, 77, 11, -100])
    for row in range(7):   # one row at a time is split, as many as `n` are not
        want_lp, want_ent, want_top, want_index = O.topk_logprobs(z[row:row + 1].double(), labels[row:row + 1], k)
        lp, ent, top, index = F.topk_logprobs_from_logits(z[row:row + 1].expand(n, v).contiguous().to(dev),
                                                          labels[row:row + 1].expand(n).to(dev), k)
        assert torch.equal(index.cpu(), want_index.expand(n, k)), row
        e = _sum_error(v) + 12 * U * 40
        _within(top, want_top.expand(n, k), e + 12 * U * want_top.abs().nan_to_num(0, 0, 0), f"top {row}")
        _within(lp, want_lp.expand(n), e + 12 * U * want_lp.abs().nan_to_num(0, 0, 0), f"logprobs {row}")
        _within(ent, want_ent.expand(n), 40 * e, f"entropy {row}")


@gpu
@pytest.mark.parametrize("n", [1, 5, 600])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_masked_throughout(dev, dtype, n):
    """A row of the type's lowest value is uniform over it, one of -inf is NaN; where a loss masks such rows out they get no gradient."""
    import verl_amd.utils.torch_functional as F
    v, k, low = 9001, 30, torch.finfo(dtype).min
    z = _logits((n, v), dtype, 2)
    z[0] = low
    if n > 1:
        z[1] = low
        z[1, 5000:] = -INF   # 5000 logits of the lowest value, the others ruled out
        z[2] = -INF
        z[3, 4:] = low
    labels = torch.full((n,), 3)
    # The outputs hold 32 bits: low / 0.7 of the types with 8 exponent bits is -4.8e38, past fp32's -3.4e38, and so -inf there.
    want = [x[:5] for x in O.topk_logprobs(z[:5].double(), labels[:5], k, 0.7)]
    want[2] = want[2].float().double()
    zd = z.to(dev).requires_grad_()
    got = F.topk_logprobs_from_logits(zd, labels.to(dev), k, 0.7)
    assert torch.equal(got[3][:5].cpu(), want[3])
    # fp16's lowest value is a number like others to the walk: of row 0 the entropy is the difference of lse and mean(z) / T, which are
    # 65504 / 0.7 = 9.4e4 both; each is off by a few of its roundings (U x 9.4e4 = 5.6e-3) and a mean by its sums' error: as above.
    reach = (z[:5].double().nan_to_num(0, 0, 0).abs().amax(-1) / 0.7) * (dtype == torch.float16)
    for a, b, name in zip(got[:3], want, ("logprobs", "entropy", "top")):
        extra = (2 * _sum_error(v) + 24 * U) * reach if name == "entropy" else 0.0
        _within(a[:5], b, 4 * (_sum_error(v) + 200 * U) + 12 * U * b.abs().nan_to_num(0, 0, 0) + extra, name)
    t, index = _teacher(_logits((n, v), torch.float32, 3), 70, 4)
    index[0, 0] = 8999
    up = torch.zeros(n)
    up[-1] = 1.0
    loss = F.topk_distillation_from_logits(zd, t.to(dev), index.to(dev), "forward_kl", temperature=0.7)
    uniform = (t[0].exp() * (t[0] + math.log(v))).sum()
    assert abs(loss[0].item() - uniform.item()) <= 20 * (_sum_error(v) + 200 * U)
    top, = torch.autograd.grad(got[2], zd, (up[:, None] * torch.ones(n, k)).to(dev), retain_graph=True)
    both = torch.autograd.grad((got[0], got[1], loss), zd, (up.to(dev),) * 3)[0]
    for d in (top, both):
        assert torch.isfinite(d).all() and (n == 1 or not d[:-1].any())
    if n == 1:   # of the uniform row: q = 1 / v
        want_d = torch.full((v,), -float(k) / v / 0.7, dtype=torch.float64)
        want_d[:k] += 1 / 0.7
        _within(top[0], want_d, HALF_STEP[dtype] * 1.01 * want_d.abs() + 4 * _sum_error(v) * k / v + 8 * U * want_d.abs()
                + torch.finfo(dtype).tiny * 2.0 ** -9, "gradient")


@gpu
@pytest.mark.parametrize("kind", ["forward_kl", "reverse_kl", "jsd"])
@pytest.mark.parametrize("k", [5, 100])
def test_rows_out_of_the_loss_get_no_gradient(dev, kind, k):
    """Rows of -inf and of NaN, whose divergence is NaN, beside rows that count: the upstream gradient decides."""
    import verl_amd.utils.torch_functional as F
    n, v = 6, 5003
    z = _logits((n, v), torch.bfloat16, 2)
    t, index = _teacher(_logits((n, v), torch.float32, 3), k, 4)
    bad = z.clone()
    bad[1], bad[4] = -INF, float("nan")
    up = torch.tensor([0.5, 0.0, -1.0, 0.0, 0.0, 2.0]).to(dev)
    grads = []
    for x in (z, bad):
        x = x.to(dev).requires_grad_()
        grads.append(torch.autograd.grad(F.topk_distillation_from_logits(x, t.to(dev), index.to(dev), kind), x, up)[0])
    assert torch.equal(*grads) and not grads[0][[1, 3, 4]].any() and grads[0][[0, 2, 5]].any()


@gpu
def test_topk_of_views_and_without_labels(dev):
    """Rows off 16 bytes, a pitch wider than the vocabulary, a transposed tensor, leading dimensions."""
    import verl_amd.utils.torch_functional as F
    base = _logits((6, 5, 3001), torch.bfloat16, 3).to(dev)
    for z in (base, base[:, :, 1:2900], base[:, 1], base.transpose(0, 1), base[..., ::2], base[0, 0]):
        lp, ent, top, index = F.topk_logprobs_from_logits(z, None, 9, 0.8)
        assert lp is None and ent.shape == z.shape[:-1] and top.shape == index.shape == (*z.shape[:-1], 9)
        flat = z.reshape(-1, z.shape[-1]).contiguous()
        _, ent2, top2, index2 = F.topk_logprobs_from_logits(flat, None, 9, 0.8)
        assert torch.equal(index.reshape(-1, 9), index2)
        for a, b in ((ent.reshape(-1), ent2), (top.reshape(-1, 9), top2)):
            assert (a - b).abs().max().item() <= 2 * _sum_error(3001) + 24 * U * 20


@gpu
def test_one_row_without_dimensions(dev):
    """A vector of logits is one row: the label and the scalars have no dimension, the alternatives one."""
    import verl_amd.utils.torch_functional as F
    z = _logits((5001,), torch.float32, 8).to(dev).requires_grad_()
    lp, ent, top, index = F.topk_logprobs_from_logits(z, torch.tensor(7, device=dev), 3)
    rows = F.topk_logprobs_from_logits(z.detach()[None], torch.tensor([7], device=dev), 3)
    assert lp.shape == ent.shape == () and top.shape == index.shape == (3,)
    for a, b in zip((lp, ent, top, index), rows):
        assert torch.equal(a, b[0])
    loss = F.topk_distillation_from_logits(z, top.detach(), index)
    assert loss.shape == () and abs(loss.item()) <= 8 * U * 30
    d, = torch.autograd.grad((lp, loss), z)
    assert d.shape == z.shape


def _gradient_bound(want, q, weight, dtype, v, reach):
    e = _sum_error(v) + 8 * U * reach
    return HALF_STEP[dtype] * want.abs() * 1.01 + 2 * e * (q * weight.abs() + want.abs()) + torch.finfo(dtype).tiny * 2.0 ** -9


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,v,k,temperature,given", [
    (3, 300, 20, 0.7, "lp ent top"), (37, 2049, 100, 1.0, "lp ent top"), (5, 33001, 64, 1.0, "top"), (4, 7, 7, 1.0, "lp"),
    (2, 70003, 256, 1.4, "ent top"), (600, 1000, 8, 1.0, "lp ent top")])
def test_topk_gradients(dev, dtype, n, v, k, temperature, given):
    import verl_amd.utils.torch_functional as F
    z, labels = _logits((n, v), dtype, 3 * n + v), _labels(n, v, n)
    labels[0] = -100
    z[n - 1, 1:min(v, 6)] = -INF
    zd = z.to(dev).requires_grad_()
    z64 = z.double().requires_grad_()
    g = torch.Generator().manual_seed(n)
    up = {"lp": torch.randn(n, generator=g), "ent": torch.randn(n, generator=g), "top": torch.randn(n, k, generator=g)}
    got = dict(zip(("lp", "ent", "top"), F.topk_logprobs_from_logits(zd, labels.to(dev), k, temperature)))
    want = dict(zip(("lp", "ent", "top"), O.topk_logprobs(z64, labels, k, temperature)))
    names = given.split()
    d, = torch.autograd.grad([got[x] for x in names], zd, [up[x].to(dev) for x in names])
    d64, = torch.autograd.grad([want[x] for x in names], z64, [up[x].double() for x in names])
    assert d.dtype == dtype and d.shape == z.shape
    q = torch.softmax(z.double() / temperature, -1)
    reach = z.double().nan_to_num(0, 0, 0).abs().amax().item() / temperature
    weight = (up["lp"].abs() + up["top"].abs().sum(1) + up["ent"].abs() * 2 * reach).double()[:, None] / temperature
    _within(d, d64, _gradient_bound(d64, q, weight, dtype, v, reach), "d_logits")


def _teacher(z, k, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    t = (z.float() + torch.randn(z.shape, generator=g)).log_softmax(-1)
    lp, index = t.topk(k, -1)
    return lp.to(dtype), index


def _check_distillation(F, dev, z, t, index, kind, beta=0.5, temperature=1.0):
    v, dtype = z.shape[-1], z.dtype
    zd = z.to(dev).requires_grad_()
    z64 = z.double().requires_grad_()
    loss = F.topk_distillation_from_logits(zd, t.to(dev), index.to(dev), kind, beta, temperature)
    want = O.topk_distillation(z64, t.double(), index.long(), kind, beta, temperature)
    assert loss.dtype == torch.float32
    with torch.no_grad():
        assert torch.equal(F.topk_distillation_from_logits(zd, t.to(dev), index.to(dev), kind, beta, temperature), loss)
    # a term is w d with w = p or q and d a difference of log-probabilities, each off by e
    log_q = torch.log_softmax(z.double() / temperature, -1)
    reach = z.double().nan_to_num(0, 0, 0).abs().amax().item() / temperature + 1
    e = _sum_error(v) + 12 * U * (reach + log_q.nan_to_num(0, 0, 0).abs().amax().item())
    counts = (index >= 0) & (index < v) & (t != -INF)
    at = torch.where(counts, index, 0).long()
    lq, tt = log_q.detach().gather(-1, at), torch.where(counts, t.double(), 0.0)
    mass = torch.where(counts, tt.exp() + lq.exp(), 0.0)
    distance = torch.where(counts, (tt - lq).abs().nan_to_num(0, 0, 0), 0.0)
    room = (mass * (e + 16 * U * distance + e * distance)).sum(-1) + 2.0 ** -126
    _within(loss, want.detach(), room, "loss")
    up = torch.randn(loss.shape, generator=torch.Generator().manual_seed(3))
    d, = torch.autograd.grad(loss, zd, up.to(dev))
    return d, up, z64, want, room, mass * (1 + distance)


def _check_distillation_gradient(F, dev, z, t, index, kind, beta=0.5, temperature=1.0):
    v, dtype = z.shape[-1], z.dtype
    d, up, z64, want, room, mass = _check_distillation(F, dev, z, t, index, kind, beta, temperature)
    d64, = torch.autograd.grad(want, z64, up.double())
    assert d.dtype == dtype and d.shape == z.shape
    q = torch.softmax(z.double() / temperature, -1)
    reach = z.double().nan_to_num(0, 0, 0).abs().amax().item() / temperature + math.log(v)
    weight = (mass.sum(-1) * up.double().abs() / temperature)[..., None]
    e = _sum_error(v) + 16 * U * reach
    at_entries = torch.zeros_like(d64).scatter_add_(-1, index.long().clamp(0, v - 1), mass * up.double().abs()[..., None] / temperature)
    bound = HALF_STEP[dtype] * 1.01 * d64.abs() + 3 * e * (q * weight + at_entries) + torch.finfo(dtype).tiny * 2.0 ** -9
    _within(d, d64, bound, "d_logits")


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype,n,v,k,temperature", [
    (torch.float32, 3, 300, 20, 0.7), (torch.bfloat16, 37, 2049, 100, 1.0), (torch.float16, 5, 33001, 64, 1.0),
    (torch.float32, 4, 7, 7, 1.0), (torch.bfloat16, 2, 70003, 256, 1.4), (torch.bfloat16, 600, 1000, 8, 1.0),
    (torch.float32, 1, 1, 1, 1.0)])
def test_distillation(dev, kind, dtype, n, v, k, temperature):
    import verl_amd.utils.torch_functional as F
    z = _logits((n, v), dtype, n + 2 * v)
    t, index = _teacher(z, k, n)
    _check_distillation_gradient(F, dev, z, t, index, kind, 0.3, temperature)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_distillation_of_padded_and_repeated_entries(dev, kind, dtype):
    """Padding by index and by log-probability, a row of nothing but padding, an index that comes several times (within and across
    blocks of 64 entries), neighbours in one lane, 16-bit log-probabilities and 32-bit indices."""
    import verl_amd.utils.torch_functional as F
    n, v, k = 6, 5003, 130
    z = _logits((n, v), dtype, 9)
    t, index = _teacher(z, k, 4, torch.bfloat16)
    index[0, 5:] = -1
    t[1, 7:] = -INF
    index[2] = -1
    t[3] = -INF
    index[4] = 17
    t[4] = t[4] - 3
    index[5] = torch.arange(k) + 2040   # both sides of a workgroup's last column
    index[1, 0], index[1, 1] = v, 2**30
    _check_distillation_gradient(F, dev, z, t, index.int(), kind)
    zd = z.to(dev).requires_grad_()
    loss = F.topk_distillation_from_logits(zd, t.to(dev), index.to(dev), kind)
    assert loss[2].item() == 0.0 and loss[3].item() == 0.0
    d, = torch.autograd.grad(loss.sum(), zd)
    assert not d[2:4].any()


@gpu
def test_distillation_where_the_student_rules_a_token_out(dev):
    """A student's logit of -inf at a teacher's token: the forward divergence is infinite, its gradient is not; the others are finite."""
    import verl_amd.utils.torch_functional as F
    z = _logits((2, 400), torch.float32, 2)
    z[:, 10] = -INF
    t = torch.tensor([[0.5, 0.25], [0.5, 0.25]]).log()
    index = torch.tensor([[10, 3], [10, 10]])
    q = torch.softmax(z.double(), -1)
    for kind in KINDS:
        zd = z.to(dev).requires_grad_()
        loss = F.topk_distillation_from_logits(zd, t.to(dev), index.to(dev), kind)
        d, = torch.autograd.grad(loss.sum(), zd)
        _within(loss, O.topk_distillation(z.double(), t.double(), index, kind), _sum_error(400) + 200 * U, kind)
        assert torch.isfinite(d).all()
        if kind == "forward_kl":
            want = 0.75 * q
            want[:, 10] = torch.tensor([-0.5, -0.75], dtype=torch.float64)
            want[0, 3] -= 0.25
            _within(d, want, 1e-5 * q + 4 * U, "gradient")


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_gradients_against_differences(dev, kind):
    """Central differences of the kernels' own losses: with steps of h the cut-off error is h^2 / 6 times a third derivative, below 1
    here for a loss below 5 at probabilities (each derivative of a softmax is a polynomial in q with coefficients up to 6), and
    the rounding error 2 x 40 u / (2 h) for losses of up to 5 made of terms of up to 8."""
    import verl_amd.utils.torch_functional as F
    n, v, k, h = 2, 24, 5, 0.03
    z = _logits((n, v), torch.float32, 12, 1.5)
    t, index = _teacher(z, k, 8)
    t, index = t.to(dev), index.to(dev)
    f = lambda x: F.topk_distillation_from_logits(x, t, index, kind, 0.4).sum()
    # (two alternatives: the third and fourth logits of the first row lie 0.012 apart, and where a step makes two of them change
    # places their log-probabilities have no derivative)
    assert (z.sort(-1, descending=True).values[:, :3].diff() < -2 * h).all()

    def top(x):
        lp, ent, two, _ = F.topk_logprobs_from_logits(x, index[:, 0].contiguous(), 2)
        return (two * torch.tensor([0.5, -0.3], device=dev)).sum() + ent.sum() + lp.sum()

    for fn in (f, top):
        zd = z.to(dev).requires_grad_()
        d, = torch.autograd.grad(fn(zd), zd)
        for j in range(0, v, 3):
            step = torch.zeros_like(z)
            step[:, j] = h
            with torch.no_grad():
                both = [fn((z + s * step).to(dev)).double().item() for s in (1, -1)]
            assert abs((both[0] - both[1]) / (2 * h) - d[:, j].sum().item()) <= n * (h * h / 6 * 6 + 80 * U / (2 * h))


@gpu
def test_a_teachers_alternatives_to_a_students_update(dev):
    """The run as it is used: the teacher's alternatives, the student's loss on them, aggregated over a mask, with its gradient."""
    import verl_amd.utils.torch_functional as F
    from verl_amd.trainer.ppo.core_algos import agg_loss
    b, l, v, k, temperature = 3, 11, 4001, 32, 1.3
    teacher, student = _logits((b, l, v), torch.bfloat16, 1), _logits((b, l, v), torch.bfloat16, 2)
    mask = (torch.arange(l)[None] < torch.tensor([11, 1, 0])[:, None]).float()
    lp, ent, top, index = F.topk_logprobs_from_logits(teacher.to(dev), _labels(b * l, v, 1).view(b, l).to(dev), k, temperature)
    x = student.to(dev).requires_grad_()
    loss = F.topk_distillation_from_logits(x, top, index, "forward_kl", temperature=temperature)
    total = agg_loss(loss, mask.to(dev), "token-mean")
    d, = torch.autograd.grad(total, x)
    x64 = student.double().requires_grad_()
    want_top, want_index = O.topk_logprobs(teacher.double(), torch.zeros(b, l, dtype=torch.int64), k, temperature)[2:]
    per_token = O.topk_distillation(x64, want_top, want_index, "forward_kl", temperature=temperature)
    want = (per_token * mask).sum() / mask.sum()
    d64, = torch.autograd.grad(want, x64)
    _within(total, want.detach(), 20 * (_sum_error(v) + 12 * U * 20), "loss")
    q = torch.softmax(student.double() / temperature, -1)
    _within(d, d64, HALF_STEP[torch.bfloat16] * 1.01 * d64.abs() + 4 * (_sum_error(v) + 400 * U) * (q + (d64.abs() > q)) / 12
            + 2.0 ** -126, "d_logits")
    assert not d[2].any()


@gpu
def test_topk_and_distillation_replay_from_a_graph(dev):
    """Captured twice, replayed on two streams at once between eager work, on new inputs."""
    import verl_amd.utils.torch_functional as F
    n, v, k = 40, 9001, 16

    def step(x, lab):
        lp, ent, top, index = F.topk_logprobs_from_logits(x, lab, k)
        loss = F.topk_distillation_from_logits(x, top.detach() - 0.1, index, "jsd", 0.3)
        d, = torch.autograd.grad((lp, ent, loss), x, (torch.ones_like(lp), torch.ones_like(ent), torch.ones_like(loss)))
        return [y.detach() for y in (lp, ent, top, index, loss, d)]

    x = _logits((n, v), torch.bfloat16, 0).to(dev).requires_grad_()
    lab = _labels(n, v, 0).to(dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, lab)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(x, lab)
        graphs.append((graph, out))
    for i in range(4):
        with torch.no_grad():
            x.copy_(_logits((n, v), torch.bfloat16, 10 + i))
            lab.copy_(_labels(n, v, 20 + i))
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for (graph, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        want = step(x, lab)
        for _, out in graphs:
            for a, b in zip(out, want):
                assert torch.equal(a, b)


@gpu
def test_capture_beside_an_eager_graph_of_the_same_leaf_is_refused(dev):
    """Autograd would wait for the eager graph's stream at the end of the captured backward pass, which ends the process."""
    import verl_amd.utils.torch_functional as F
    x = _logits((4, 300), torch.float32, 0).to(dev).requires_grad_()
    t, index = x.detach().log_softmax(-1).topk(5, -1)
    for fn in (lambda: F.topk_logprobs_from_logits(x, None, 5)[2], lambda: F.topk_distillation_from_logits(x, t, index)):
        alive = fn()
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="eager graph"):
            with torch.cuda.graph(graph):
                torch.ones(1, device=dev)
                fn()
        torch.cuda.synchronize()
        del alive
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            elsewhere = fn()   # on a stream that can join a capture
        torch.cuda.current_stream().wait_stream(side)
        for kept in (elsewhere, None):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                fn()
            torch.cuda.synchronize()
            elsewhere = kept = None


@gpu
def test_topk_on_another_stream_and_twice(dev):
    """The same call gives the same bits, on a stream of its own too; a second backward pass over a kept graph as well."""
    import verl_amd.utils.torch_functional as F
    z, labels = _logits((30, 70001), torch.float32, 6).to(dev).requires_grad_(), _labels(30, 70001, 6).to(dev)
    first = F.topk_logprobs_from_logits(z, labels, 50)
    g = [torch.ones_like(first[0]), torch.ones_like(first[1]), torch.ones_like(first[2])]
    d = torch.autograd.grad(first[:3], z, g, retain_graph=True)[0]
    assert torch.equal(torch.autograd.grad(first[:3], z, g)[0], d)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        second = F.topk_logprobs_from_logits(z, labels, 50)
    torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(first, second):
        assert torch.equal(a, b)


@gpu
def test_what_autograd_is_refused(dev):
    import verl_amd.utils.torch_functional as F
    z = _logits((4, 300), torch.float32, 1).to(dev)
    t, index = _teacher(z.cpu(), 5, 1)
    t, index, lab = t.to(dev), index.to(dev), torch.zeros(4, dtype=torch.int64, device=dev)
    calls = (lambda x: F.topk_logprobs_from_logits(x, lab, 5)[2].sum(), lambda x: F.topk_distillation_from_logits(x, t, index).sum())
    for fn in calls:
        x = z.clone().requires_grad_()
        d, = torch.autograd.grad(fn(x) ** 2, x, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            d.sum().backward()
        with pytest.raises(NotImplementedError, match="forward mode"), torch.autograd.forward_ad.dual_level():
            fn(torch.autograd.forward_ad.make_dual(z, torch.ones_like(z)))
        with pytest.raises(RuntimeError):
            torch.vmap(fn)(z[None])
        with pytest.raises(RuntimeError, match="torch.jit.trace"):
            torch.jit.trace(fn, (z,), check_trace=False)
        x = z.clone().requires_grad_()
        y = fn(x)
        with torch.no_grad():
            x.add_(1.0)
        with pytest.raises(RuntimeError, match="inplace"):
            y.backward()
        with torch.autograd.graph.save_on_cpu():
            x = z.clone().requires_grad_()
            y = fn(x)
        assert torch.equal(torch.autograd.grad(y, x)[0], torch.autograd.grad(fn(x), x)[0])


@gpu
def test_refusals_with_gpu_tensors(dev):
    import verl_amd.utils.torch_functional as F
    z = _logits((4, 300), torch.float32, 1).to(dev)
    lab = torch.zeros(4, dtype=torch.int64, device=dev)
    for k in (0, -1, 257, 301):
        with pytest.raises(AssertionError, match="k must be"):
            F.topk_logprobs_from_logits(z, lab, k)
    with pytest.raises(AssertionError, match="k must be"):
        F.topk_logprobs_from_logits(z[:, :10], lab, 11)
    with pytest.raises(AssertionError, match="k must be an int"):
        F.topk_logprobs_from_logits(z, lab, 2.0)
    for temperature in (0.0, -1.0, INF, NAN):
        with pytest.raises(AssertionError, match="temperature"):
            F.topk_logprobs_from_logits(z, lab, 2, temperature)
    with pytest.raises(AssertionError, match="labels"):
        F.topk_logprobs_from_logits(z, lab[:3], 2)
    with pytest.raises(AssertionError, match="whole numbers"):
        F.topk_logprobs_from_logits(z, lab.float(), 2)
    with pytest.raises(AssertionError, match="fp32, bf16 or fp16"):
        F.topk_logprobs_from_logits(z.double(), lab, 2)
    with pytest.raises(AssertionError):
        F.topk_logprobs_from_logits(z[:0], lab[:0], 2)
    t, index = z[:, :5].contiguous(), torch.zeros(4, 5, dtype=torch.int64, device=dev)
    for bad in ((t[:3], index[:3]), (t[:, :4], index), (t[0], index[0]), (t[None], index[None])):
        with pytest.raises(AssertionError, match="teacher"):
            F.topk_distillation_from_logits(z, *bad)
    with pytest.raises(AssertionError, match="int64 or int32"):
        F.topk_distillation_from_logits(z, t, index.float())
    with pytest.raises(AssertionError, match="1 to 256"):
        F.topk_distillation_from_logits(z, z[:, :257].contiguous(), torch.zeros(4, 257, dtype=torch.int64, device=dev))
    with pytest.raises(AssertionError, match="1 to 256"):
        F.topk_distillation_from_logits(z, t[:, :0], index[:, :0])


def test_refusals_on_the_host():
    """What needs no GPU to be refused: tensors on the CPU, unknown divergences, a weight outside (0, 1), and by the C interface
    sizes, options, alignments and workspaces."""
    import verl_amd.utils.torch_functional as F
    from verl_amd import _cabi
    z, lab = torch.zeros(4, 300), torch.zeros(4, dtype=torch.int64)
    t, index = torch.zeros(4, 5), torch.zeros(4, 5, dtype=torch.int64)
    with pytest.raises(AssertionError, match="must live on the GPU"):
        F.topk_logprobs_from_logits(z, lab, 5)
    with pytest.raises(AssertionError, match="must live on the GPU"):
        F.topk_distillation_from_logits(z, t, index)
    with pytest.raises(ValueError, match="Invalid divergence"):
        F.topk_distillation_from_logits(z, t, index, "kl")
    for beta in (0.0, 1.0, -0.5, NAN):
        with pytest.raises(AssertionError, match="beta"):
            F.topk_distillation_from_logits(z, t, index, "jsd", beta)
    lib, at = _cabi.lib(), 4096   # never read
    topk = lambda logits=at, dtype=0, n=4, v=300, ld=300, labels=at, k=5, rcp=1.0, lp=at, top=at, index=at, stats=at, ws=at, size=1 << 30: \
        lib.vamd_row_topk(logits, dtype, n, v, ld, labels, k, rcp, lp, at, top, index, stats, ws, size, None)
    for bad in (dict(logits=None), dict(dtype=3), dict(n=0), dict(v=0), dict(ld=299), dict(labels=None), dict(k=0), dict(k=257),
                dict(k=301, v=300), dict(rcp=0.0), dict(rcp=-1.0), dict(rcp=INF), dict(rcp=NAN), dict(top=None), dict(index=None),
                dict(stats=at + 4), dict(v=1 << 31, ld=1 << 31), dict(n=1 << 31)):
        assert topk(**bad) == -1, bad
    need = lib.vamd_row_topk_workspace_bytes(1, 151936, 1, 20)
    assert need > 0 and lib.vamd_row_topk_workspace_bytes(4096, 151936, 1, 20) == 0
    assert topk(dtype=1, n=1, v=151936, ld=151936, k=20, size=need - 1) == -2
    assert topk(dtype=1, n=1, v=151936, ld=151936, k=20, ws=None) == -2
    div = lambda kind=0, beta=0.5, teacher=at, index=at, loss=at, k=5, stats=at, entries=at, size=1 << 30: lib.vamd_row_divergence(
        at, 0, 4, 300, 300, teacher, index, k, kind, beta, 1.0, loss, stats, entries, size, None)
    for bad in (dict(kind=3), dict(kind=-1), dict(kind=2, beta=1.0), dict(kind=2, beta=NAN), dict(teacher=None), dict(index=None),
                dict(loss=None), dict(k=0), dict(k=257), dict(stats=at + 8), dict(stats=None), dict(entries=None)):
        assert div(**bad) == -1, bad
    for k in (5, 65):
        assert div(k=k, size=lib.vamd_row_divergence_entries_bytes(4, 300, 0, k) - 1) == -2
    other, need = 1 << 20, lib.vamd_row_topk_backward_workspace_bytes(4, 300, 0, 5)
    back = lambda labels=at, index=at, stats=at, lp=at, ent=None, top=None, out=other, ld=300, ws=at, size=need: \
        lib.vamd_row_topk_backward(at, 0, 4, 300, 300, labels, 5, index, 1.0, stats, lp, ent, top, out, ld, ws, size, None)
    div_back = lambda index=at, k=5, stats=at, entries=at, d_loss=at, out=other, ld=300: lib.vamd_row_divergence_backward(
        at, 0, 4, 300, 300, index, k, 1.0, stats, entries, d_loss, out, ld, None)
    for bad in (dict(out=None), dict(out=at), dict(ld=299), dict(stats=None), dict(stats=at + 4)):   # at: the logits themselves
        assert back(**bad) == -1 and div_back(**bad) == -1, bad
    assert back(lp=None) == -1 and back(labels=None) == -1 and back(lp=None, top=at, index=None) == -1
    assert div_back(index=None) == -1 and div_back(entries=None) == -1 and div_back(d_loss=None) == -1 and div_back(k=257) == -1
    assert back(size=need - 1) == -2 and back(ws=None) == -2
