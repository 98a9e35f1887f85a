"""The categorical readout against plain 64-bit implementations of its formulas.

Tolerances, with e = 2^-24 (half a step of f32) and h = half a step of the output type:
  product   the integer sum is exact; its conversion to f32, the two scales and the bias are one rounding each: 4 e of the
            largest intermediate, then h of the result.
  rules     at most one rounding each for the repetition, the frequency's product, two subtractions and the biases.
  draw      indices: equal.  Scores are compared in f64 on both sides.
  distill   z = beta l carries e |z|; the difference to the maximum another; the exponential 3 e; a sum of n terms over at least 256
            threads n/256 + 16 roundings: so lse (and a relative error of q) is within E = e (n / 256 + 32 + 4 max|z|); the listed
            entries add e (top + 16 + 4 max|t|) relative on p, and the loss sums top terms.
"""
import math

import numpy as np
import pytest
import torch

import fullsize_checks as F

pytestmark = pytest.mark.gpu

E = 2.0**-24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["f32", "bf16", "f16"]
TINY = {torch.float32: 2.0**-149, torch.bfloat16: 2.0**-133, torch.float16: 2.0**-24}  # subnormal steps


def half(t):
    return torch.finfo(t).eps / 2


def gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def spaced(x, pitch, shift):
    """x's values in rows `pitch` apart that start `shift` elements behind a 256-byte boundary, and the buffer around them."""
    space = torch.full((x.shape[0] * pitch + shift + 16,), 77, dtype=x.dtype, device=x.device)
    view = space[shift:shift + x.shape[0] * pitch].view(x.shape[0], pitch)[:, :x.shape[1]]
    view.copy_(x)
    return view, space


def near(got, want, tol):
    """Within tol elementwise; infinities and NaN in the same places."""
    got, want = got.double(), want.double()
    assert got.shape == want.shape
    same = (got == want) | (got.isnan() & want.isnan())
    # Every number within the tolerance is as good as the value; from (2 - 2^-24) 2^127 on, f32 rounds them to infinity.
    same |= got.isinf() & (got.sign() == want.sign()) & (want.abs() + tol >= (2 - 2.0**-24) * 2.0**127)
    ok = same | ((got - want).abs() <= tol)
    assert bool(ok.all()), f"{int((~ok).sum())} values, worst {((got - want).abs() / tol)[~ok].max()} tolerances off"


# ---- 8-bit rows and the product


def quantised(x):
    """(q, scale) by the definition: the scale in f32 (divided in 64 bits, since torch divides f32 by a number through its
    reciprocal), the quotient in 64 bits."""
    scale = (x.double().abs().amax(1) / 127).float().double()
    q = (x.double() / scale[:, None]).nan_to_num(0.0, posinf=0.0, neginf=0.0).round().clamp(-127, 127)
    return q, scale


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("rows, cols, pitch, shift", [(1, 1, 1, 0), (3, 7, 9, 1), (2, 16, 16, 0), (5, 129, 131, 3), (4, 784, 784, 0), (33, 1000, 1008, 8), (2, 16385, 16387, 5), (1, 40000, 40000, 0),
                                                      (700, 64, 64, 0)])
def test_quantize_rows(T, dtype, rows, cols, pitch, shift):
    x = (torch.randn(rows, cols, generator=gen(rows * cols), device="cuda") * 5).to(dtype)
    x[0, cols // 2] = 0
    x[-1] = x[-1] * 0 if rows > 2 else x[-1]  # a row of zeros
    v, _ = spaced(x, pitch, shift)
    q, scale = T.quantize_rows(v)
    want, s = quantised(x)
    assert torch.equal(scale.double(), s) and torch.equal(q.double(), want) and q.dtype == torch.int8


def test_quantize_rows_at_the_borders(T):
    """Quotients that lie on a half, or next to one, and rows whose scale is subnormal."""
    rows = []
    for top in (127.0, 1.27, 3e-3, 127 * 2.0**-140, 1e-40, 3e-43, 2.0**-149, 3e38):
        scale = np.float32(top) / np.float32(127)
        with np.errstate(all="ignore"):
            halves = ((np.arange(-127, 127) + 0.5).astype(np.float64) * np.float64(scale)).astype(np.float32)
            rows.append(np.concatenate([[np.float32(top)], halves, np.nextafter(halves, np.float32(np.inf)), np.nextafter(halves, np.float32(-np.inf))]).clip(-top, top))
    x = torch.from_numpy(np.stack(rows).astype(np.float32)).cuda()
    q, scale = T.quantize_rows(x)
    s64 = (np.abs(x.cpu().numpy()).max(1) / np.float32(127)).astype(np.float64)
    assert np.array_equal(scale.cpu().numpy().astype(np.float64), s64)
    with np.errstate(all="ignore"):
        want = np.clip(np.rint(x.cpu().numpy().astype(np.float64) / s64[:, None]), -127, 127)
    want[s64 == 0] = 0
    assert np.array_equal(q.cpu().numpy(), want)


def test_quantize_rows_with_infinities(T):
    x = torch.ones(4, 33, device="cuda")
    x[0, 5], x[1, 32], x[2, 0] = math.inf, math.nan, -math.inf
    q, scale = T.quantize_rows(x)
    assert scale[0] == math.inf and scale[1].isnan() and scale[2] == math.inf and scale[3] == torch.tensor(1.0) / 127
    assert not q[:3].any() and bool((q[3] == 127).all())
    y = T.int8_matmul(q, scale, T.align_rows_int8(torch.ones(3, 33, dtype=torch.int8, device="cuda")), torch.ones(3, device="cuda"))
    assert y[:3].isnan().all() and y[3].isfinite().all()


def product64(q, qs, w, ws, b, dtype):
    acc = q.double() @ w.double().T
    y = acc * qs.double()[:, None] * ws.double()
    z = y if b is None else y + b.double()
    return z, 4 * E * (y.abs() + z.abs()) + half(dtype) * z.abs() + TINY[dtype]


SHAPES = [(1, 1, 1), (1, 16, 17), (2, 128, 127), (1, 4096, 129), (16, 784, 300), (17, 31, 128), (31, 513, 1000), (33, 784, 4097), (64, 1024, 640), (65, 256, 257), (127, 2049, 130), (128, 128, 128),
          (129, 300, 385), (257, 130, 1025), (511, 1000, 77), (513, 4096, 513), (1000, 96, 2000), (2049, 333, 515), (5000, 200, 700), (6300, 130, 761), (3000, 1030, 1500)]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("m, k, n", SHAPES)
def test_int8_matmul(T, dtype, m, k, n):
    g = gen(m + k + n)
    a = T.align_rows_int8(torch.randint(-128, 128, (m, k), generator=g, device="cuda", dtype=torch.int8))
    w = T.align_rows_int8(torch.randint(-128, 128, (n, k), generator=g, device="cuda", dtype=torch.int8))
    qs, ws = torch.rand(m, generator=g, device="cuda") * 1e-3, torch.rand(n, generator=g, device="cuda") * 1e-2
    b = torch.randn(n, generator=g, device="cuda") if (m + n) % 2 else None
    space = torch.full((m + 2, n + 3), 55.0, dtype=dtype, device="cuda")
    out = T.int8_matmul(a, qs, w, ws, b, out=space[1:m + 1, 1:n + 1])
    want, tol = product64(a, qs, w, ws, b, dtype)
    near(out, want, tol)
    space[1:m + 1, 1:n + 1] = 55.0  # nothing around the output was written
    assert bool((space == 55.0).all())
    assert torch.equal(T.int8_matmul(a, qs, w, ws, b, out_dtype=dtype), T.int8_matmul(a, qs, w, ws, b, out_dtype=dtype))


def test_int8_matmul_is_exact_to_the_largest_sums(T):
    """Sums past 2^24: their conversion to f32 is the only rounding."""
    k = 131071
    a = T.align_rows_int8(torch.full((2, k), -128, dtype=torch.int8, device="cuda"))
    w = T.align_rows_int8(torch.full((3, k), -128, dtype=torch.int8, device="cuda"))
    w[1] = 127
    w[2, ::2] = 1
    one = torch.ones(3, device="cuda")
    got = T.int8_matmul(a, one[:2], w, one)
    want = (a.double() @ w.double().T).float()
    assert torch.equal(got, want) and float(want[0, 0]) == float(np.float32(128 * 128 * k))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("m, k, n", [(1, 4096, 513), (5, 33, 40), (33, 784, 4097), (300, 1111, 520), (1030, 640, 300)])
def test_int8_linear(T, dtype, m, k, n):
    g = gen(m * k + n)
    x, _ = spaced((torch.randn(m, k, generator=g, device="cuda") * 3).to(dtype), k + 5, 3)
    w = T.align_rows_int8(torch.randint(-127, 128, (n, k), generator=g, device="cuda", dtype=torch.int8))
    ws, b = torch.rand(n, generator=g, device="cuda") * 1e-2, torch.randn(n, generator=g, device="cuda")
    out = T.int8_linear(x, w, ws, b)
    q, s = quantised(x)
    want, tol = product64(q, s, w, ws, b, dtype)
    near(out, want, tol)
    q8, s8 = T.quantize_rows(x)
    assert torch.equal(out, T.int8_matmul(q8, s8, w, ws, b, out_dtype=dtype))
    wq, wsc = T.quantize_rows(torch.randn(n, k, generator=g, device="cuda"))  # a layer's weights by channel
    q64 = wq.double() * wsc.double()[:, None]
    near(T.int8_linear(x, wq, wsc, out_dtype=torch.float32), (q * s[:, None]) @ q64.T, 8 * E * (q * s[:, None]).abs() @ q64.abs().T + 1e-30)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("m, k, n", [(1, 8, 1), (1, 4096, 513), (2, 4096, 4096), (16, 512, 300), (3, 24, 40), (1, 8192, 130), (8, 1000, 77), (5, 136, 20000), (7, 128, 129)])
def test_int8_linear_of_few_tokens(T, dtype, m, k, n):
    """Small products quantise their tokens themselves: what the two calls give, rows of zeros and of infinities among them."""
    g = gen(m * k + n)
    x = (torch.randn(m, k, generator=g, device="cuda") * torch.logspace(-3, 3, m, device="cuda")[:, None]).to(dtype)
    if m > 2:
        x[1] = 0
        x[2, k // 2] = math.inf
    w, ws = T.quantize_rows(torch.randn(n, k, generator=g, device="cuda"))
    b = torch.randn(n, generator=g, device="cuda")
    q, s = T.quantize_rows(x)
    for out_dtype in TYPES:
        got, want = T.int8_linear(x, w, ws, b, out_dtype=out_dtype), T.int8_matmul(q, s, w, ws, b, out_dtype=out_dtype)
        assert torch.equal(got.nan_to_num(12345.0), want.nan_to_num(12345.0)) and bool((got.isnan() == want.isnan()).all())
    if m > 2:
        assert got[2].isnan().all() and torch.equal(got[1], b.to(out_dtype))


# ---- rules


def adjust64(x, rules):
    """Row by row, in 64 bits; (result, magnitude of what was rounded on the way)."""
    out, mag = x.double().clone().cpu().numpy(), x.double().abs().cpu().numpy().copy()
    mag[~np.isfinite(mag)] = 0
    r, v = out.shape
    c = {k: (t.cpu().numpy() if isinstance(t, torch.Tensor) else t) for k, t in rules.items()}
    for i in range(r):
        if c.get("history") is not None:
            h = c["history"][c["history_ptr"][i]:c["history_ptr"][i + 1]].astype(np.int64)
            n_prompt = max(int(c["n_prompt"][i]), 0) if c.get("n_prompt") is not None else 0
            seen = np.bincount(h[(h >= 0) & (h < v)], minlength=v)
            told = h[n_prompt:]
            told = np.bincount(told[(told >= 0) & (told < v)], minlength=v)
            rep = float(c["repetition"][i]) if c.get("repetition") is not None else 1.0
            fr = float(c["frequency"][i]) if c.get("frequency") is not None else 0.0
            pr = float(c["presence"][i]) if c.get("presence") is not None else 0.0
            hit = seen > 0
            out[i] = np.where(hit, np.where(out[i] > 0, out[i] / rep, out[i] * rep), out[i])
            mag[i] += np.where(np.isfinite(out[i]), np.abs(out[i]), 0) + abs(fr) * told + abs(pr) * (told > 0)
            out[i] = np.where(told > 0, out[i] - fr * told - pr, out[i])
        if c.get("bias_ids") is not None:
            for e in range(c["bias_ptr"][i], c["bias_ptr"][i + 1]):
                if 0 <= c["bias_ids"][e] < v:
                    out[i, c["bias_ids"][e]] += float(c["bias_values"][e])
                    if np.isfinite(c["bias_values"][e]):
                        mag[i, c["bias_ids"][e]] += abs(float(c["bias_values"][e]))
        if c.get("mask") is not None:
            m = int(c["mask_rows"][i]) if c.get("mask_rows") is not None else i
            if 0 <= m < c["mask"].shape[0]:
                bits = np.unpackbits(np.ascontiguousarray(c["mask"][m]).view(np.uint8), bitorder="little")[:v]
                out[i][bits == 0] = -np.inf
    return torch.from_numpy(out).cuda(), torch.from_numpy(mag).cuda()


def make_rules(r, v, seed, hist=40, biases=6, masks=2, index=torch.int32):
    g = gen(seed)
    rnd = lambda *s: torch.rand(*s, generator=g, device="cuda")  # noqa: E731
    whole = lambda lo, hi, *s: torch.randint(lo, hi, s, generator=g, device="cuda")  # noqa: E731
    rules = {}
    if hist:
        lengths = whole(0, hist + 1, r)
        lengths[0] = 0  # a row that has seen nothing
        rules["history_ptr"] = torch.cat([lengths.new_zeros(1), lengths.cumsum(0)])
        rules["history"] = ((rnd(max(int(lengths.sum()), 1)) ** 2 * (v + 2)).long() - 1).to(index)  # -1 and v are padding
        rules["n_prompt"] = (lengths * rnd(r) * 1.3).int()
        rules["repetition"], rules["frequency"], rules["presence"] = 0.8 + rnd(r), rnd(r) - 0.3, rnd(r)
        rules["repetition"][-1] = 1.0
    if biases:
        rules["bias_ids"] = whole(-1, v + 1, r, biases).sort(1)[0].int().reshape(-1)
        rules["bias_values"] = torch.randn(r * biases, generator=g, device="cuda")
        rules["bias_ptr"] = torch.arange(r + 1, device="cuda") * biases
    if masks:
        rules["mask"] = whole(-(1 << 31), 1 << 31, masks, (v + 31) // 32 + 1).int()
        rules["mask_rows"] = whole(-1, masks + 1, r).int()  # -1 and `masks` say none
    return rules


def check_adjust(T, x, rules, dtype, **kw):
    got = T.adjust_logits(x, **rules, **kw)
    want, mag = adjust64(x, rules)
    near(got, want, 12 * E * mag + half(dtype) * want.abs().nan_to_num(0, 0, 0) + TINY[dtype])
    return got


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("r, v, hist, biases, masks", [(1, 1, 3, 1, 1), (1, 2, 0, 0, 1), (3, 31, 5, 0, 0), (4, 33, 40, 6, 2), (2, 8191, 300, 50, 1), (3, 8193, 2000, 50, 3), (1, 50001, 300, 5, 1),
                                                       (5, 16400, 0, 300, 0), (7, 20000, 5000, 0, 2), (2, 131073, 9000, 40, 1), (300, 70, 30, 3, 4)])
def test_adjust_logits(T, dtype, r, v, hist, biases, masks):
    x = (torch.randn(r, v, generator=gen(r + v), device="cuda") * 4).to(dtype)
    check_adjust(T, x, make_rules(r, v, r * v, hist, biases, masks, torch.int64 if v % 2 else torch.int32), dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("pitch, shift", [(1000, 0), (1007, 1), (1005, 7), (1016, 8)])
def test_adjust_logits_strides_and_in_place(T, dtype, pitch, shift):
    x = (torch.randn(5, 1000, generator=gen(pitch), device="cuda") * 4).to(dtype)
    rules = make_rules(5, 1000, pitch)
    want = T.adjust_logits(x, **rules)
    v, space = spaced(x, pitch, shift)
    to, around = spaced(x, 1000 + shift, 3)
    assert torch.equal(T.adjust_logits(v, **rules, out=to), want) and torch.equal(v, x)
    assert T.adjust_logits(v, **rules, out=v) is v and torch.equal(v, want)
    v.fill_(77), to.fill_(77)
    assert bool((space == 77).all()) and bool((around == 77).all())


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_adjust_logits_odd_values(T, dtype):
    """Infinities, NaN, the type's lowest value and signed zeros, penalised, biased and masked; a mask that leaves nothing."""
    v = 70
    x = torch.zeros(4, v, device="cuda", dtype=dtype)
    low = torch.finfo(dtype).min
    x[:, 0], x[:, 1], x[:, 2], x[:, 3], x[:, 4] = math.inf, -math.inf, math.nan, low, -0.0
    rules = dict(history=torch.arange(8, device="cuda").repeat(4), history_ptr=torch.arange(5, device="cuda") * 8, n_prompt=torch.tensor([0, 8, 3, 99], device="cuda", dtype=torch.int32),
                 repetition=torch.tensor([1.5, 0.5, 1.0, 2.0], device="cuda"), frequency=torch.full((4,), 0.5, device="cuda"), presence=torch.full((4,), 0.25, device="cuda"),
                 bias_ids=torch.tensor([5, 5, 5, 6, 3, 60], device="cuda", dtype=torch.int32), bias_values=torch.tensor([1.0, 2.0, -0.5, -math.inf, 1.0, math.inf], device="cuda"),
                 bias_ptr=torch.tensor([0, 4, 4, 6, 6], device="cuda"), mask=torch.zeros(4, 3, device="cuda", dtype=torch.int32))
    rules["mask"][1:3] = -1
    rules["mask"][3] = 0b100
    got = T.adjust_logits(x, **rules)
    want, _ = adjust64(x, rules)
    want = want.to(torch.float32).to(dtype).double()  # an f16 beyond the range becomes an infinity
    near(got, want, 4 * half(dtype) * want.abs().nan_to_num(0, 0, 0) + TINY[dtype])
    assert bool((got[0] == -math.inf).all()) and got[3, 2].isnan() and bool((got[3, :2] == -math.inf).all())


def test_adjust_logits_counts_past_16_bits(T):
    n = 70000
    x = torch.ones(1, 9, device="cuda")
    history = torch.full((n,), 4, device="cuda", dtype=torch.int32)
    got = T.adjust_logits(x, history=history, history_ptr=torch.tensor([0, n], device="cuda"), n_prompt=torch.tensor([1000], device="cuda", dtype=torch.int32),
                          frequency=torch.tensor([0.5], device="cuda"))
    assert float(got[0, 4]) == 1 - 0.5 * 69000 and bool((got[0, :4] == 1).all())


def test_adjust_logits_without_rules_copies(T):
    x = torch.randn(3, 100, device="cuda")
    assert torch.equal(T.adjust_logits(x), x)
    assert T.adjust_logits(x[:0]).shape == (0, 100)
    rules = dict(history=torch.zeros(0, device="cuda", dtype=torch.int32), history_ptr=torch.zeros(4, device="cuda", dtype=torch.int64), repetition=torch.full((3,), 2.0, device="cuda"))
    assert torch.equal(T.adjust_logits(x, **rules), x)


# ---- the draw


def uniforms(rows, cols, key, offset=0):
    k = np.arange(cols, dtype=np.uint64)
    row = (np.arange(rows, dtype=np.uint64) + np.uint64(offset))[:, None]
    words = F._philox(row, np.uint64(0), k >> np.uint64(2), 0x44524157, np.uint64(key & 0xFFFFFFFF), np.uint64(key >> 32))
    words = np.stack(np.broadcast_arrays(*words))  # [4][rows][cols]
    w = np.take_along_axis(words, np.broadcast_to((k & np.uint64(3)).astype(np.int64), words.shape[1:])[None], 0)[0]
    return ((w >> np.uint64(9)).astype(np.float64) + 0.5) * 2.0**-23


def draw64(x, u, beta):
    l = x.double().cpu().numpy()
    out = []
    for i in range(l.shape[0]):
        b = 1.0 if beta is None else float(beta[i])
        with np.errstate(all="ignore"):
            s = l[i] if b == math.inf else b * l[i] - np.log(-np.log(np.float64(u[i])))
        s = np.where((l[i] > -math.inf) & (s > -math.inf), s, -math.inf)
        out.append(-1 if not b >= 0 or not (s > -math.inf).any() else int(np.argmax(s)))
    return torch.tensor(out)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("r, v, pitch, shift", [(1, 1, 1, 0), (3, 2, 2, 0), (5, 5, 7, 1), (4, 63, 64, 0), (2, 2047, 2048, 0), (3, 2049, 2051, 3), (1, 50001, 50001, 0), (2, 131072, 131072, 0),
                                                (600, 33, 33, 0), (9, 20000, 20008, 8)])
def test_draw_categories(T, dtype, r, v, pitch, shift):
    g = gen(r * v)
    x, _ = spaced((torch.randn(r, v, generator=g, device="cuda") * 3).masked_fill_(torch.rand(r, v, generator=g, device="cuda") < 0.2, -math.inf).to(dtype), pitch, shift)
    beta = torch.rand(r, generator=g, device="cuda") * 2
    beta[::3] = math.inf
    for key, offset in ((0, 0), (0xFEDCBA9876543210, 5), (12345, (1 << 32) - r)):
        u = uniforms(r, v, key, offset)
        assert torch.equal(T.draw_categories(x, key, beta=beta, row_offset=offset).cpu(), draw64(x, u, beta))
    assert torch.equal(T.draw_categories(x, 12345, row_offset=(1 << 32) - r).cpu(), draw64(x, u, None))
    noise, _ = spaced(torch.from_numpy(u).float().cuda(), v + 3, 1)
    assert torch.equal(T.draw_categories(x, 1, beta=beta, noise=noise).cpu(), draw64(x, noise.cpu().numpy(), beta))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_draw_categories_odd_rows(T, dtype):
    v = 3001
    x = torch.zeros(10, v, device="cuda", dtype=dtype)
    x[0] = -math.inf
    x[1] = -math.inf
    x[1, 2999] = torch.finfo(dtype).min  # the one category left
    x[2] = math.nan
    x[3, 7] = x[3, 9] = math.inf
    x[4, 11] = math.nan
    x[5] = torch.finfo(dtype).min
    x[6, 5:9] = 2.0
    x[8] = torch.finfo(dtype).max
    beta = torch.tensor([1.0, 1.0, 1.0, 1.0, math.inf, 1.0, math.inf, -1.0, 1.0, math.nan], device="cuda")
    u = uniforms(10, v, 99)
    got = T.draw_categories(x, 99, beta=beta).cpu()
    assert torch.equal(got, draw64(x, u, beta))
    assert got[0] == -1 and got[1] == 2999 and got[2] == -1 and got[3] == 7 and got[6] == 5 and got[7] == -1 and got[9] == -1


def test_draw_categories_ties_and_noise_at_the_ends(T):
    """Equal scores go to the lowest category wherever they lie; noise 1 wins, noise 0 never does, noise that is no number is passed over."""
    for v in (8, 4096, 100000):
        x = torch.zeros(3, v, device="cuda")
        noise = torch.full((3, v), 0.25, device="cuda")
        noise[1, v - 1] = noise[1, v // 2] = 1.0
        noise[2] = 0.0
        noise[2, 5], noise[2, 6] = math.nan, 1e-30
        assert T.draw_categories(x, 0, noise=noise).tolist() == [0, v // 2, 6]


def test_draw_categories_near_ties(T):
    """Scores that f32 cannot tell apart are drawn as 64 bits order them."""
    v = 5000
    g = gen(3)
    u = torch.rand(200, v, generator=g, device="cuda").clamp_(1e-3, 0.999)
    x = ((-u.double().log()).log() + 3.0).float()  # every score within about 1e-7 of 3
    assert torch.equal(T.draw_categories(x, 0, noise=u).cpu(), draw64(x, u.cpu().numpy(), None))


def test_draw_categories_frequencies(T):
    """Chances follow the softmax: 40000 rows of the same four logits, five standard deviations."""
    x = torch.tensor([[0.0, 1.0, -math.inf, 2.0]], device="cuda").repeat(40000, 1)
    got = torch.bincount(T.draw_categories(x, T.RngKey(7)), minlength=4).double().cpu() / 40000
    p = x[0].double().softmax(0).cpu()
    assert bool(((got - p).abs() <= 5 * (p * (1 - p) / 40000).sqrt()).all()) and got[2] == 0


# ---- distillation


def distill64(x, ids, teacher, beta, weight):
    """(loss, lse, grad, tolerance of loss, of lse, of grad before its rounding)"""
    z = x.double() * float(np.float32(beta))
    r, v = z.shape
    there = (ids >= 0) & (ids < v) & (teacher.double() != -math.inf)
    at = ids.long().clamp(0, v - 1)
    t = torch.where(there, teacher.double() * float(np.float32(beta)), -math.inf)
    some = there.any(1)
    w = torch.ones(r, device="cuda", dtype=torch.float64) if weight is None else weight.double()
    live = some & (w != 0)
    log_p = torch.where(there, t - t.logsumexp(1, keepdim=True), -math.inf)
    p = log_p.exp()
    lse = z.logsumexp(1)
    empty = lse == -math.inf
    q = torch.where(empty[:, None], 0.0, (z - lse[:, None]).exp())
    term = torch.where(p > 0, p * (log_p - (z.gather(1, at) - lse[:, None])), 0.0)
    loss = torch.where(empty, math.inf, term.sum(1))
    grad = (w * float(np.float32(beta)))[:, None] * q.clone().scatter_add_(1, at, -p)
    fine = lambda a: a.abs().nan_to_num(0, 0, 0)  # noqa: E731
    zmax, tmax, top = fine(z).amax(1), fine(t).amax(1) if t.shape[1] else fine(lse) * 0, ids.shape[1]
    e_lse = E * (v / 256 + 32 + 4 * zmax + fine(lse))
    e_p = E * (top + 16 + 4 * tmax)
    sizes = (p * (fine(log_p) + fine(z.gather(1, at)) + fine(lse)[:, None] + 1)).sum(1)
    e_loss = e_lse + (e_p + E * (top + 8)) * sizes
    e_grad = (w * beta).abs()[:, None] * (q * (2 * e_lse + E * (4 * zmax + 8))[:, None] + torch.zeros_like(q).scatter_add_(1, at, p * e_p[:, None]) + 4 * E * q)
    dead = ~live
    loss, lse, grad = loss.masked_fill(dead, 0), lse.masked_fill(dead, 0), grad.masked_fill(dead[:, None], 0)
    return loss, lse, grad, e_loss, e_lse, e_grad


def check_distill(T, x, ids, teacher, beta, weight):
    dtype = x.dtype
    loss, lse = T.distill_loss(x, ids, teacher, beta=beta, weight=weight)
    grad = T.distill_grad(x, lse, ids, teacher, beta=beta, weight=weight)
    loss2, grad2 = T.distill_step(x, ids, teacher, beta=beta, weight=weight)
    L, S, G, el, es, eg = distill64(x, ids, teacher, beta, weight)
    assert grad.dtype == grad2.dtype == dtype and loss.dtype == lse.dtype == torch.float32
    near(loss, L, el + E * L.abs().nan_to_num(0, 0, 0))
    near(lse, S, es + E * S.abs().nan_to_num(0, 0, 0))
    near(loss2, L, el + E * L.abs().nan_to_num(0, 0, 0))
    for got in (grad, grad2):
        near(got, G, eg + half(dtype) * (G.abs().nan_to_num(0, 0, 0) + eg.nan_to_num(0, 0, 0)) + TINY[dtype])
    return loss, lse, grad


def make_distill(r, v, top, seed, dtype, teacher_dtype=torch.float32, index=torch.int32):
    g = gen(seed)
    x = (torch.randn(r, v, generator=g, device="cuda") * 3).to(dtype)
    ids = torch.randint(-1, v + 1, (r, top), generator=g, device="cuda").to(index)  # -1 and v are not listed; the same id comes twice
    teacher = (torch.randn(r, top, generator=g, device="cuda") * 3).to(teacher_dtype)
    weight = torch.rand(r, generator=g, device="cuda") - 0.3
    weight[::4] = 0
    return x, ids, teacher, weight


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("r, v, top", [(1, 1, 1), (2, 2, 3), (3, 33, 4), (5, 1000, 64), (4, 1000, 1024), (9, 8193, 7), (2, 32768, 100), (3, 50001, 33), (1, 131072, 128), (2, 200003, 20), (1, 500001, 9),
                                       (1, 1000003, 5), (700, 130, 6)])
def test_distill(T, dtype, r, v, top):
    x, ids, teacher, weight = make_distill(r, v, top, r * v + top, dtype, TYPES[v % 3], torch.int64 if top % 2 else torch.int32)
    check_distill(T, x, ids, teacher, 0.5, None)
    check_distill(T, x, ids, teacher, 1.3, weight)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("v, pitch, shift", [(1000, 1000, 0), (999, 1007, 1), (1000, 1005, 7), (40000, 40008, 8), (40001, 40003, 1)])
def test_distill_strides(T, dtype, v, pitch, shift):
    x, ids, teacher, weight = make_distill(6, v, 17, pitch, dtype)
    loss, grad = T.distill_step(x, ids, teacher, beta=0.7, weight=weight)
    xs, space = spaced(x, pitch, shift)
    is_, _ = spaced(ids, 19, 1)
    ts, _ = spaced(teacher, 21, 3)
    to, around = spaced(x, v + shift + 1, 2)
    loss2, lse = T.distill_loss(xs, is_, ts, beta=0.7, weight=weight)
    L, S, G, el, es, eg = distill64(x, ids, teacher, 0.7, weight)
    near(loss2, L, el + E * L.abs())
    for got in (T.distill_grad(xs, lse, is_, ts, beta=0.7, weight=weight, out=to), T.distill_step(xs, is_, ts, beta=0.7, weight=weight, out=to)[1], grad):
        near(got, G, eg + half(dtype) * (G.abs() + eg) + TINY[dtype])
    assert torch.equal(xs, x)
    xs.fill_(77), to.fill_(77)
    assert bool((space == 77).all()) and bool((around == 77).all())


@pytest.mark.parametrize("v", [40, 3001, 140000])
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_distill_odd_rows(T, dtype, v):
    """Padding rows full of NaN, rows that list nothing, masked categories, rows with nothing left, the type's lowest value."""
    x, ids, teacher, _ = make_distill(9, v, 6, v, dtype)
    ids = (torch.arange(6, device="cuda") * 5)[None].repeat(9, 1).int()
    weight = torch.ones(9, device="cuda")
    x[0], weight[0] = math.nan, 0
    ids[1] = -1
    teacher[2] = -math.inf
    x[3, ::2] = -math.inf  # ids 0, 10, 20 are masked: the loss is infinite, the gradient is not
    x[4] = -math.inf
    x[5, 1:] = torch.finfo(dtype).min
    ids[6] = 7  # one category six times
    x[7, 20:] = -math.inf  # a few categories left
    ids[7, 4:] = -1
    teacher[8, 1:] = -math.inf
    L, S, G, el, es, eg = distill64(x, ids, teacher, 1.0, weight)
    loss, lse, grad = check_distill(T, x, ids, teacher, 1.0, weight)
    assert loss[0] == 0 and not grad[0].any() and loss[1] == 0 and not grad[1:3].any() and loss[3] == math.inf and loss[4] == math.inf
    assert lse[4] == -math.inf and bool(grad[4].isfinite().all()) and bool(grad[3].isfinite().all())


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("v", [7, 3000, 70001])
def test_distill_rows_of_the_lowest_value(T, dtype, v):
    """A mask of the type's lowest value that leaves nothing is a uniform row; one that leaves two equal categories, a half each."""
    x = torch.full((3, v), torch.finfo(dtype).min, device="cuda", dtype=dtype)
    x[1, 2] = x[1, v - 1] = 1.5
    x[2] = torch.finfo(dtype).max
    x[2, ::2] = torch.finfo(dtype).min
    ids = torch.tensor([[1, 3, 5]], device="cuda").repeat(3, 1)
    ids[1] = torch.tensor([2, 2, v - 1])
    teacher = torch.tensor([[0.5, -1.0, 2.0]], device="cuda").repeat(3, 1)
    for beta in (0.5, 1.0, 2.0):
        p = (teacher.double() * beta).softmax(1)
        q = torch.zeros(3, v, device="cuda", dtype=torch.float64)
        q[0], q[1, 2], q[1, v - 1] = 1 / v, 0.5, 0.5
        q[2, 1::2] = 1 / (v // 2)
        want_loss = (p * (p.log() - q.gather(1, ids).log())).sum(1)
        want = beta * q.scatter_add(1, ids, -p)
        loss, lse = T.distill_loss(x, ids, teacher, beta=beta)
        near(loss, want_loss, E * 64 * (1 + want_loss.abs()))
        for grad in (T.distill_grad(x, lse, ids, teacher, beta=beta), T.distill_step(x, ids, teacher, beta=beta)[1]):
            rows = (0, 1, 2) if dtype != torch.float16 else (1, )  # f16's ends are ordinary numbers: lse holds the row's size to 2^-8 only
            for i in rows:
                near(grad[i], want[i], half(dtype) * want[i].abs() + E * 64 * beta + TINY[dtype])


@pytest.mark.parametrize("rows", [3, 700])  # few rows: one launch; many: the lists in their own
@pytest.mark.parametrize("top", [1, 33, 64, 65, 129, 1024])
@pytest.mark.parametrize("several", [1, 3, 40, 1000])
def test_distill_categories_listed_again(T, rows, top, several):
    """Lists that take up few categories again and again, in every order, with entries that are not listed among them."""
    v = 2003
    x, _, teacher, weight = make_distill(rows, v, top, rows + top, torch.bfloat16)
    g = gen(several)
    of = torch.randint(0, v, (rows, several), generator=g, device="cuda")
    ids = of.gather(1, torch.randint(0, several, (rows, top), generator=g, device="cuda"))
    ids[torch.rand(rows, top, generator=g, device="cuda") < 0.1] = -1
    loss, lse, grad = check_distill(T, x, ids, teacher, 0.8, weight)
    again = T.distill_loss(x, ids, teacher, beta=0.8, weight=weight)[0], T.distill_grad(x, lse, ids, teacher, beta=0.8, weight=weight)
    assert torch.equal(loss, again[0]) and torch.equal(grad, again[1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("top", [6, 70])
def test_distill_odd_rows_among_many(T, dtype, top):
    """The odd rows again, where the lists have a launch of their own."""
    n, v = 900, 1031
    x, ids, teacher, _ = make_distill(n, v, top, top, dtype)
    weight = torch.ones(n, device="cuda")
    x[0::9], weight[0::9] = math.nan, 0
    ids[1::9] = -1
    teacher[2::9] = -math.inf
    x[3::9, ::2] = -math.inf
    x[4::9] = -math.inf
    x[5::9, 1:] = torch.finfo(dtype).min
    ids[6::9] = 7
    x[7::9, 20:] = -math.inf
    ids[7::9] = ids[7::9] % 20
    teacher[8::9, 1:] = -math.inf
    loss, lse, grad = check_distill(T, x, ids, teacher, 1.0, weight)
    assert not loss[0::9].any() and not grad[0::9].any() and not grad[1::9].any() and not grad[2::9].any() and bool((lse[4::9] == -math.inf).all())
    assert bool(grad[4::9].isfinite().all())


def test_distill_nan_stays_in_its_row(T):
    x, ids, teacher, _ = make_distill(4, 5000, 5, 1, torch.float32)
    ids = ids.clamp(0, 4999)
    x[1, 4321] = math.nan
    x[2, 17] = math.inf
    loss, grad = T.distill_step(x, ids, teacher)
    assert loss[1].isnan() and loss[2].isnan() and loss[0].isfinite() and loss[3].isfinite() and grad[0].isfinite().all() and grad[3].isfinite().all()


def test_distill_gradient_against_differences(T):
    """(loss(z + d) - loss(z - d)) / 2d with d = 2^-5: d^2 / 6 times the third derivative (at most beta^3 / 6 < 1 here) and twice the
    loss's error over 2 d."""
    v, d = 24, 2.0**-5
    x, ids, teacher, _ = make_distill(1, v, 5, 4, torch.float32)
    ids = torch.tensor([[3, 9, 9, 20, -1]], device="cuda")
    _, grad = T.distill_step(x, ids, teacher, beta=1.25)
    plus = x + d * torch.eye(v, device="cuda")
    minus = x - d * torch.eye(v, device="cuda")
    every = lambda a: T.distill_loss(a, ids.repeat(v, 1), teacher.repeat(v, 1), beta=1.25)[0].double()  # noqa: E731
    _, _, _, el, _, _ = distill64(x, ids, teacher, 1.25, None)
    near(((every(plus) - every(minus)) / (2 * d))[None], grad, d * d / 6 * 1.25**3 + float(el[0]) * 2 / d + E * 16)


def test_distill_weight_comes_from_above(T):
    """distill_grad takes any weight for the same lse: the gradient is linear in it."""
    x, ids, teacher, _ = make_distill(4, 3000, 8, 9, torch.float32)
    ids = ids.clamp(0, 2999)
    _, lse = T.distill_loss(x, ids, teacher)
    one = T.distill_grad(x, lse, ids, teacher)
    w = torch.tensor([2.0, -4.0, 0.0, 0.5], device="cuda")
    assert torch.equal(T.distill_grad(x, lse, ids, teacher, weight=w), one * w[:, None] + 0.0)


# ---- together, streams, graphs


def chain(T, s):
    logits = T.int8_linear(s["x"], s["w"], s["ws"], s["b"])
    T.adjust_logits(logits, **s["rules"], out=logits)
    drawn = T.draw_categories(logits, 42, beta=s["beta"])
    loss, grad = T.distill_step(logits, s["ids"], s["teacher"], beta=0.5)
    return logits, drawn, loss, grad


def make_chain(T, seed, m=6, k=200, n=3000):
    g = gen(seed)
    s = dict(x=torch.randn(m, k, generator=g, device="cuda", dtype=torch.bfloat16), ws=torch.rand(n, generator=g, device="cuda") * 1e-3, b=torch.randn(n, generator=g, device="cuda"))
    s["w"] = T.align_rows_int8(torch.randint(-127, 128, (n, k), generator=g, device="cuda", dtype=torch.int8))
    s["rules"] = make_rules(m, n, seed)
    s["beta"] = torch.ones(m, device="cuda")
    _, s["ids"], s["teacher"], _ = make_distill(m, n, 9, seed, torch.bfloat16)
    return s


def test_the_operators_together(T):
    s = make_chain(T, 5)
    logits, drawn, loss, grad = chain(T, s)
    plain = T.int8_linear(s["x"], s["w"], s["ws"], s["b"])
    want, mag = adjust64(plain, s["rules"])
    near(logits, want, 12 * E * mag + half(torch.bfloat16) * want.abs().nan_to_num(0, 0, 0))
    assert torch.equal(drawn.cpu(), draw64(logits, uniforms(6, 3000, 42), s["beta"]))
    L, _, G, el, _, eg = distill64(logits, s["ids"], s["teacher"], 0.5, None)
    near(loss, L, el + E * L.abs().nan_to_num(0, 0, 0))
    near(grad, G, eg + half(torch.bfloat16) * (G.abs() + eg))


def test_on_another_stream_and_in_two_graphs(T):
    """The same results on a side stream, and from two captured graphs replayed in turn and at once with new inputs in place."""
    sets = [make_chain(T, 11), make_chain(T, 12)]
    want = [chain(T, s) for s in sets]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = chain(T, sets[0])
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    graphs, outs, ins = [], [], []
    for i in range(2):
        ins.append({k: v.clone() if isinstance(v, torch.Tensor) and k != "w" else v for k, v in sets[i].items()})
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(chain(T, ins[i]))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for i in (0, 1):
            streams[i].wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in (0, 1):
            assert all(torch.equal(a, b) for a, b in zip(outs[i], want[i]))
    ins[0]["x"].copy_(sets[0]["x"] * 2)
    graphs[0].replay()
    fresh = chain(T, {**sets[0], "x": sets[0]["x"] * 2})
    assert all(torch.equal(a, b) for a, b in zip(outs[0], fresh))


def test_offsets_past_32_bits(T):
    """Rows 2^30 + 16 elements apart: the third begins past 2^31."""
    v, pitch = 5000, (1 << 30) + 16
    space = torch.empty(2 * pitch + v, dtype=torch.bfloat16, device="cuda")
    far = space.as_strided((3, v), (pitch, 1))
    x = torch.randn(3, v, generator=gen(1), device="cuda").bfloat16()
    far.copy_(x)
    rules, beta = make_rules(3, v, 1), torch.ones(3, device="cuda")
    _, ids, teacher, _ = make_distill(3, v, 7, 1, torch.bfloat16)
    assert torch.equal(T.draw_categories(far, 3, beta=beta), T.draw_categories(x, 3, beta=beta))
    q, s = T.quantize_rows(x)
    assert all(torch.equal(a, b) for a, b in zip(T.quantize_rows(far), (q, s)))
    loss, grad = T.distill_step(x, ids, teacher)
    loss2, grad2 = T.distill_step(far, ids, teacher)
    assert torch.equal(loss, loss2) and torch.equal(grad, grad2)
    want = T.adjust_logits(x, **rules)
    T.adjust_logits(far, **rules, out=far)
    assert torch.equal(far, want)
    lse = T.distill_loss(x, ids, teacher)[1]
    T.distill_grad(x, lse, ids, teacher, out=far)
    near(far, grad, 4 * half(torch.bfloat16) * grad.abs().double() + 1e-6)
    w, ws = T.quantize_rows(torch.randn(v, v, generator=gen(2), device="cuda"))
    T.int8_matmul(q, s, w, ws, out=far)
    assert torch.equal(far, T.int8_matmul(q, s, w, ws, out_dtype=torch.bfloat16))
    many = torch.randn(700, v, generator=gen(3), device="cuda").bfloat16()  # the kernel of many tokens, a column per 2^22 elements
    wide = torch.empty(700 * (1 << 22), dtype=torch.bfloat16, device="cuda").as_strided((700, v), (1 << 22, 1))
    T.int8_linear(many, w, ws, out=wide)
    assert torch.equal(wide, T.int8_linear(many, w, ws))


def test_ids_past_32_bits_are_padding(T):
    x = torch.randn(2, 300, generator=gen(1), device="cuda")
    h = torch.tensor([5, (1 << 40) + 5, -(1 << 40) + 7, 1 << 32, 8, 5], device="cuda")
    rules = dict(history=h, history_ptr=torch.tensor([0, 6, 6], device="cuda"), frequency=torch.ones(2, device="cuda"))
    clean = dict(rules, history=torch.tensor([5, 8, 5], device="cuda"), history_ptr=torch.tensor([0, 3, 3], device="cuda"))
    assert torch.equal(T.adjust_logits(x, **rules), T.adjust_logits(x, **clean))
    ids = torch.tensor([[3, (1 << 40) + 3, -1]], device="cuda").repeat(2, 1)
    teacher = torch.zeros(2, 3, device="cuda")
    a, b = T.distill_step(x, ids, teacher), T.distill_step(x, ids[:, :1], teacher[:, :1])
    assert all(torch.equal(i, j) for i, j in zip(a, b))


def test_current_device_and_errors_stay_the_callers(T):
    """A refused call leaves no error behind, and the current device does not change."""
    before = torch.cuda.current_device()
    x = torch.randn(4, 100, device="cuda")
    with pytest.raises(T.ThrmlError):
        T.draw_categories(x, 1, row_offset=1 << 33)
    T.draw_categories(x, 1)
    assert torch.cuda.current_device() == before and bool((x + 1).isfinite().all())


def test_context_reports_no_wait_that_ran_out(T):
    from thrml_rs_b200 import engine
    q, s = T.quantize_rows(torch.randn(70, 300, device="cuda"))
    T.int8_matmul(q, s, q, s)
    torch.cuda.synchronize()
    engine.default_context(0).synchronize()  # would raise THRML_ERR_TIMEOUT


def test_refused_on_the_gpu(T):
    x = torch.zeros(4, 64, device="cuda")
    w = torch.zeros(8, 64, dtype=torch.int8, device="cuda")
    one = torch.ones(8, device="cuda")
    bad = [
        lambda: T.quantize_rows(x.T), lambda: T.quantize_rows(x.double()), lambda: T.quantize_rows(x[0]), lambda: T.quantize_rows(x[:1].expand(4, 64)),
        lambda: T.int8_linear(x, w[:, :32], one), lambda: T.int8_linear(x, w, one[:3]), lambda: T.int8_linear(x, w, None), lambda: T.int8_linear(x, w, one.cpu()),
        lambda: T.int8_linear(x, w, one, out_dtype=torch.int32), lambda: T.int8_linear(x, w, one, out=torch.zeros(4, 9, device="cuda")),
        lambda: T.int8_linear(x[:, :40], torch.zeros(8, 40, dtype=torch.int8, device="cuda"), one),
        lambda: T.int8_matmul(x, one, w, one), lambda: T.int8_matmul(w[:, 1:33], one, w[:, 1:33], one),
        lambda: T.adjust_logits(x, history=torch.zeros(3, device="cuda", dtype=torch.int32)), lambda: T.adjust_logits(x, repetition=one[:4]),
        lambda: T.adjust_logits(x, mask=torch.zeros(4, 1, device="cuda", dtype=torch.int32)), lambda: T.adjust_logits(x, mask=torch.zeros(3, 2, device="cuda", dtype=torch.int32)),
        lambda: T.adjust_logits(x, bias_ids=torch.zeros(3, device="cuda", dtype=torch.int32)), lambda: T.adjust_logits(x, mask_rows=torch.zeros(4, device="cuda", dtype=torch.int32)),
        lambda: T.draw_categories(x, -1), lambda: T.draw_categories(x, 1 << 64), lambda: T.draw_categories(x, 1, beta=one), lambda: T.draw_categories(x, 1, noise=x[:, :9]),
        lambda: T.draw_categories(x, 1, out=torch.zeros(4, device="cuda")), lambda: T.draw_categories(x, 1, row_offset=1 << 32),
        lambda: T.distill_loss(x, x.int(), x[:, :3]), lambda: T.distill_loss(x, x, x), lambda: T.distill_step(x, x.int(), x, beta=0), lambda: T.distill_step(x, x.int(), x, weight=one),
        lambda: T.distill_grad(x, one, x.int(), x), lambda: T.distill_step(x, x.int(), x, out=x.half()), lambda: T.distill_step(x, x.int(), x, out=x),
    ]
    for f in bad:
        with pytest.raises(T.ThrmlError):
            f()


def test_no_rows(T):
    x, i = torch.zeros(0, 64, device="cuda"), torch.zeros(0, 3, device="cuda", dtype=torch.int32)
    w = torch.zeros(8, 64, dtype=torch.int8, device="cuda")
    assert T.quantize_rows(x)[0].shape == (0, 64) and T.int8_linear(x, w, torch.ones(8, device="cuda")).shape == (0, 8)
    assert T.int8_linear(torch.zeros(2, 64, device="cuda"), w[:0], torch.ones(0, device="cuda")).shape == (2, 0)
    assert T.draw_categories(x, 1).shape == (0,) and T.distill_step(x, i, x[:, :3])[1].shape == (0, 64)
    y = torch.randn(3, 64, device="cuda")  # rows that list nothing
    none = torch.zeros(3, 0, device="cuda")
    loss, grad = T.distill_step(y, none.int(), none)
    assert not loss.any() and not grad.any()
