"""The categorical readout at the ends of its range: logits and temperatures far from 1, outputs and inputs in odd places.

Tolerances of the distillation, with e = 2^-24, h = half a step of the output type, n categories, and everything relative to the
row's largest beta l (d = the distance to it from a category's, which the kernels form by subtracting first, so that the size of the logits
does not count):
  q      (l - ref) b2 carries 4 e of the exponent: two roundings of b2 (the constant and the product), one of the difference, one of the
         product or multiply-add; the reference lies within the row's spread s of what counts.  The exponential is within 4 e, a sum of n
         terms over at least 256 threads n / 256 + 16 roundings, log2 of it (at most 30) with its rounding 32.  So E = e (n / 256 + 64 + 8 (d + s))
         relative; where that nears 1 the probability is below 2^-126 and counts as 0.
  p      the same over the listed: e (top + 16 + 8 (distance + spread)).
  loss   per listed entry three sums of numbers no larger than |log p| + d + log n + s.
  lse    one multiply-add more: e of its size.  distill_grad has the rounding of an lse of at most 2^8 besides.
"""
import math

import pytest
import torch

from test_gpu_readout import adjust64, E, IDS, TINY, TYPES, draw64, gen, half, near, uniforms  # noqa: F401

pytestmark = pytest.mark.gpu


def fine(a):
    return a.nan_to_num(0, 0, 0)


def distill64(x, ids, teacher, beta):
    """(loss, lse, gradient for weight 1, their tolerances, what an lse that is given adds to the last) from 64-bit differences."""
    l, t = x.double(), teacher.double()
    n, top = x.shape[1], ids.shape[1]
    high = l.amax(1, keepdim=True)
    d = fine(beta * (high - l)).clamp_(max=1e4)  # beyond, probabilities are 0 in 64 bits too
    s = torch.where(d < 70, d, 0.0).amax(1, keepdim=True)
    e = torch.where(l == high, 1.0, (beta * (l - high)).exp())
    total = e.sum(1, keepdim=True)
    q = e / total
    there = (ids >= 0) & (ids < n) & (t != -math.inf)
    at = ids.long().clamp(0, n - 1)
    t = torch.where(there, t, -math.inf)
    t_high = t.amax(1, keepdim=True)
    t = torch.where(t == t_high, 0.0, beta * (t - t_high))
    t = torch.where(there, t, -math.inf)
    log_p = t - t.exp().sum(1, keepdim=True).log()
    p = log_p.exp()
    z = beta * (l.gather(1, at) - high)
    loss = torch.where(p > 0, p * (log_p - z + total.log()), 0.0).sum(1)
    lse = beta * high[:, 0] + total[:, 0].log()
    grad = beta * q.clone().scatter_add_(1, at, -p)
    d_p = fine(-t).clamp(max=1e4)
    e_sum = E * (n / 256 + 64 + 8 * s[:, 0])
    e_q = e_sum[:, None] + 8 * E * d
    e_p = E * (top + 16 + 8 * (d_p + torch.where(d_p < 70, d_p, 0.0).amax(1, keepdim=True)))
    size = p * (fine(log_p.abs()) + fine(z.abs()) + math.log(n) + s + 1)
    e_loss = e_sum + ((e_p + 8 * E) * size).sum(1) + E * loss.abs()
    e_lse = e_sum + 2 * E * lse.abs()
    e_grad = beta * (q * e_q + torch.zeros_like(q).scatter_add_(1, at, p * e_p)) + 4 * E * (grad.abs() + beta * q) + beta * 2.0**-125
    given = 2 * E * lse.abs() * (lse.abs() <= 260)  # a smaller lse is taken as it is, with its rounding
    return loss, lse, grad, e_loss, e_lse, e_grad, given[:, None] * beta * q


def check_large(T, x, ids, teacher, beta, times):
    """Loss, then gradient, and the step, on `times` copies of the rows."""
    dtype, r = x.dtype, x.shape[0]
    L, S, G, el, es, eg, given = distill64(x, ids, teacher, float(torch.tensor(beta, dtype=torch.float32)))
    rep = lambda a: a.repeat(times, *[1] * (a.dim() - 1))  # noqa: E731
    xs, is_, ts = rep(x), rep(ids), rep(teacher)
    loss, lse = T.distill_loss(xs, is_, ts, beta=beta)
    grad = T.distill_grad(xs, lse, is_, ts, beta=beta)
    loss2, grad2 = T.distill_step(xs, is_, ts, beta=beta)
    # Copies may differ in their last bits: they start at different places of 16 bytes, so their sums have other orders.
    for i in {0, times // 2, times - 1}:
        mine = slice(i * r, (i + 1) * r)
        near(lse[mine], S, es)
        near(loss[mine], L, el)
        near(loss2[mine], L, el)
        for g, more in ((grad2, 0.0), (grad, given)):
            near(g[mine], G, eg + more + half(dtype) * (G.abs() + eg + more) + TINY[dtype])


def large_rows(size, n, dtype, seed):
    """A row that is all +-size; two categories of it beside -inf; half of it one and half the other; a few steps of the type around it."""
    g = gen(seed)
    x = torch.full((5, n), size, device="cuda", dtype=torch.float32)
    x[1] = -size
    x[2] = -math.inf
    x[2, n // 2] = x[2, n - 1] = -size
    x[3, ::2] = -size
    x[4] = size * (1 - 2 * half(dtype) * torch.randint(0, 4, (n,), generator=g, device="cuda"))
    return x.to(dtype)


SIZES = [60.0, 200.0, 300.0, 1e4, 65504.0, 1e6, 1e9, 1e10, 1e15, 1e20, 1e30, 3e38]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("beta", [0.5, 0.7, 1.0])
@pytest.mark.parametrize("n, times", [(7, 1), (3000, 1), (70001, 1), (7, 400), (3001, 90)])
def test_distill_large_logits(T, dtype, beta, n, times):
    """Rows of large logits that leave something: what their mask's fill is does not matter."""
    for size in SIZES:
        if size > torch.finfo(dtype).max:
            continue
        x = large_rows(size, n, dtype, n)
        ids = torch.tensor([[n - 1, n // 2, 0, -1, 1]], device="cuda").repeat(5, 1)
        ids[2, 2:] = -1  # the two that are left
        teacher = torch.tensor([[0.5, -1.0, 2.0, 9.0, 0.25]], device="cuda").repeat(5, 1)
        check_large(T, x, ids, teacher, beta, times)


@pytest.mark.parametrize("dtype", TYPES[:2], ids=IDS[:2])
@pytest.mark.parametrize("beta", [2.0**-100, 1e-10, 1e10, 2.0**100])
@pytest.mark.parametrize("times", [1, 200])
def test_distill_ends_of_beta(T, dtype, beta, times):
    x = (torch.randn(4, 1001, generator=gen(2), device="cuda") * 3).to(dtype)
    x[2] *= 1e30
    ids = torch.arange(5, device="cuda")[None].repeat(4, 1) * 9
    check_large(T, x, ids, torch.zeros(4, 5, device="cuda"), beta, times)


@pytest.mark.parametrize("times", [1, 300])
def test_distill_padding_has_no_lse(T, times):
    """Rows of weight 0 are not read, whatever their lse is."""
    x = torch.randn(4 * times, 999, generator=gen(3), device="cuda")
    ids, teacher = torch.arange(3, device="cuda")[None].repeat(4 * times, 1), torch.zeros(4 * times, 3, device="cuda")
    weight = torch.tensor([1.0, 0.0, 0.0, 0.0], device="cuda").repeat(times)
    lse = T.distill_loss(x, ids, teacher, weight=weight)[1]
    want = T.distill_grad(x, lse, ids, teacher, weight=weight)
    lse = lse.view(times, 4)
    lse[:, 1], lse[:, 2], lse[:, 3] = math.nan, math.inf, 1e30
    x.view(times, 4, -1)[:, 1:] = math.nan
    assert torch.equal(T.distill_grad(x, lse.reshape(-1), ids, teacher, weight=weight), want) and not want.view(times, 4, -1)[:, 1:].any()


@pytest.mark.parametrize("beta", [0.5, 0.7, 1.0, 2.0])
@pytest.mark.parametrize("times", [1, 120])
def test_distill_large_teacher_logits(T, beta, times):
    """The teacher's logits likewise: entries a few steps apart at any size, and a list that is all the lowest value."""
    n = 3000
    x = torch.randn(4, n, generator=gen(1), device="cuda")
    ids = torch.arange(9, device="cuda")[None].repeat(4, 1) * 7
    for size in SIZES + [torch.finfo(torch.float32).max]:
        t = torch.full((4, 9), -size, device="cuda")
        t[1] = size * (1 - 2 * half(torch.float32) * torch.arange(9, device="cuda"))
        t[2, ::2] = size
        t[3] = -t[1]
        check_large(T, x, ids, t, beta, times)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("beta", [1e30, 1e38, 2.3e38, 2.4e38, torch.finfo(torch.float32).max])
@pytest.mark.parametrize("r, v", [(3, 5), (4, 3001), (2, 131072), (700, 40)])
def test_draw_categories_large_beta(T, dtype, beta, r, v):
    """Temperatures next to 0: the largest logit wins, among log-probabilities, positive logits and both; -infinity is masked."""
    x = torch.randn(r, v, generator=gen(v), device="cuda") * 3
    x[0] = x[0].log_softmax(0)  # every product with beta may overflow, or none
    x[-1] = x[-1].abs().neg() * 0.1
    x[1, ::3] = -math.inf
    x = x.to(dtype)
    b = torch.full((r,), beta, device="cuda")
    assert torch.equal(T.draw_categories(x, 77, beta=b).cpu(), draw64(x, uniforms(r, v, 77), b))
    noise = torch.rand(r, v, generator=gen(9), device="cuda").clamp_(1e-6, 0.999999)
    assert torch.equal(T.draw_categories(x, 77, beta=b, noise=noise).cpu(), draw64(x, noise.cpu().numpy(), b))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_outputs_beside_inputs_and_over_them(T, dtype):
    """Columns of one buffer may hold input and output side by side; an output that shares elements with an input is refused."""
    both = torch.randn(6, 2048, generator=gen(4), device="cuda").to(dtype)
    x, y = both[:, :1024], both[:, 1024:]
    w, ws = T.quantize_rows(torch.randn(1024, 1024, generator=gen(5), device="cuda"))
    ids, teacher = torch.arange(4, device="cuda")[None].repeat(6, 1), torch.zeros(6, 4, device="cuda")
    beta = torch.ones(6, device="cuda")
    mask = torch.full((6, 32), 0x55555555, dtype=torch.int32, device="cuda")
    for f in (lambda o: T.int8_linear(x, w, ws, out=o), lambda o: T.adjust_logits(x, mask=mask, out=o), lambda o: T.distill_step(x, ids, teacher, out=o)[1],
              lambda o: T.distill_grad(x, beta, ids, teacher, out=o)):
        want = f(None)
        assert f(y) is y and torch.equal(y, want)
        for o in (both[:, 1:1025], both[:, 1023:2047], both.view(-1)[8:8 + 6 * 1024].view(6, 1024)):
            with pytest.raises(T.ThrmlError, match="overlap"):
                f(o)
    for f in (lambda: T.int8_linear(x, w, ws, out=x), lambda: T.distill_step(x, ids, teacher, out=x), lambda: T.distill_grad(x, beta, ids, teacher, out=x)):
        with pytest.raises(T.ThrmlError):
            f()


@pytest.mark.parametrize("offset", [-1, (1 << 32) - 3, 1 << 63, 1 << 64, (1 << 64) + 5, -(1 << 64)])
def test_draw_categories_refuses_offsets_of_any_size(T, offset):
    with pytest.raises(T.ThrmlError, match="row_offset"):
        T.draw_categories(torch.zeros(4, 64, device="cuda"), 1, row_offset=offset)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_adjust_logits_any_repetition(T, dtype):
    """Penalties from the smallest to the largest: the reciprocal of many of them is no f32, their quotients are."""
    reps = torch.tensor([2.0**-149, 2.0**-140, 1e-39, 2.0**-126, 1e-3, 1.0, 7.0, 1e30, 1e38, 3e38], device="cuda")
    n = 64
    x = torch.logspace(-40, 38, n, device="cuda")[None].repeat(10, 1)
    x[:, ::3] *= -1
    x = x.clamp(torch.finfo(dtype).min, torch.finfo(dtype).max).to(dtype)
    rules = dict(history=torch.arange(n, device="cuda").repeat(10), history_ptr=torch.arange(11, device="cuda") * n, repetition=reps)
    got = T.adjust_logits(x, **rules)
    want, _ = adjust64(x, rules)
    want = want.float().to(dtype).double()  # one rounding to f32 and one to the type: beyond their range an infinity
    near(got, want, (2 * E + 2 * half(dtype)) * want.abs().nan_to_num(0, 0, 0) + TINY[dtype])


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("n, times, top", [(3001, 90, 70), (9001, 100, 129), (140003, 20, 40)])
def test_distill_large_logits_with_lists(T, dtype, n, times, top):
    """Lists of a warp, of four, and rows of several CTAs, whose sums a gradient forms again."""
    g = gen(top)
    for size in (300.0, 1e4, 1e9, 1e30):
        if size > torch.finfo(dtype).max:
            continue
        x = large_rows(size, n, dtype, n)
        ids = torch.randint(-1, n + 1, (5, top), generator=g, device="cuda")
        ids[2] = torch.tensor([n // 2, n - 1], device="cuda").repeat(top)[:top]
        check_large(T, x, ids, torch.randn(5, top, generator=g, device="cuda"), 0.7, times)


@pytest.mark.parametrize("dtype, n, rows", [(torch.float32, 1048601, 1), (torch.float32, 1048601, 40), (torch.bfloat16, 4500001, 2), (torch.float16, 2097200, 38), (torch.float32, 1048601, 100)])
def test_distill_rows_beyond_4_mb(T, dtype, n, rows):
    """Where sums are formed again, by each of a gradient's CTAs or, for many such rows, shared: ordinary rows, a large one among them, one of
    the lowest value."""
    x = torch.randn(rows, n, generator=gen(6), device="cuda") * 3
    x[-1] = torch.finfo(dtype).min
    if rows > 1:
        x[0] += 1000
    x = x.to(dtype)
    ids = torch.randint(0, n, (rows, 6), generator=gen(7), device="cuda")
    ids[:, 3] = n - 1
    teacher = torch.randn(rows, 6, generator=gen(8), device="cuda")
    loss, lse = T.distill_loss(x, ids, teacher, beta=0.5)
    grad = T.distill_grad(x, lse, ids, teacher, beta=0.5)
    loss2, grad2 = T.distill_step(x, ids, teacher, beta=0.5)
    for i in {0, rows // 2, rows - 1}:
        one = slice(i, i + 1)
        L, S, G, el, es, eg, given = distill64(x[one], ids[one], teacher[one], 0.5)
        near(lse[one], S, es)
        near(loss[one], L, el)
        near(loss2[one], L, el)
        for got, more in ((grad2, 0.0), (grad, given)):
            near(got[one], G, eg + more + half(dtype) * (G.abs() + eg + more) + TINY[dtype])
