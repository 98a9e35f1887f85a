"""The categorical readout's operators as a user calls them, with their plain forms: the 8-bit product, the rules on logits,
the draw of a category and the distillation loss.  A case says its operator, its sizes and its types; `prepare` makes the
inputs on the GPU, `run` makes one pass."""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
TAG_DRAW = 0x44524157


def listed():
    return [
        # one token through a square layer: the weights' bytes are all there is to do, latency counts
        {"name": "linear one token", "op": "linear", "m": 1, "k": 4096, "n": 4096, "type": "bf16", "bias": False},
        # a short ragged batch into an odd number of channels, 784 inputs (an image's pixels)
        {"name": "linear ragged batch", "op": "linear", "m": 33, "k": 784, "n": 4097, "type": "f32", "bias": True},
        # serving: 64 sequences, the logits of 65536 categories
        {"name": "linear readout", "op": "linear", "m": 64, "k": 4096, "n": 65536, "type": "f16", "bias": False},
        # a batch of long prompts (or 8192 chains' features) through a wide layer
        {"name": "linear prompt", "op": "linear", "m": 8192, "k": 4096, "n": 16384, "type": "bf16", "bias": True},
        # one sequence of a few hundred tokens, an odd number of categories
        {"name": "adjust one row", "op": "adjust", "r": 1, "v": 50001, "type": "f32", "history": 300, "biases": 5, "masks": 1},
        # serving: 256 sequences with a few thousand tokens each, a grammar's masks shared among them
        {"name": "adjust batch", "op": "adjust", "r": 256, "v": 131072, "type": "bf16", "history": 4096, "biases": 64, "masks": 16},
        # few sequences with long contexts
        {"name": "adjust long history", "op": "adjust", "r": 16, "v": 32768, "type": "f16", "history": 60000, "biases": 300, "masks": 0},
        # the smallest draw, with uniforms that the caller gives (a parity run)
        {"name": "draw given noise", "op": "draw", "r": 4, "v": 1009, "type": "f32", "noise": True},
        # serving: 256 sequences, noise from the key
        {"name": "draw batch", "op": "draw", "r": 256, "v": 131072, "type": "bf16", "noise": False},
        # few rows of a small model, forward then backward
        {"name": "distill few rows", "op": "distill", "r": 33, "v": 5003, "top": 8, "type": "f32", "step": False},
        # a training step's rows, loss and gradient in one call
        {"name": "distill step", "op": "distill", "r": 4096, "v": 32768, "top": 64, "type": "bf16", "step": True},
        # many categories, the loss first and the gradient later
        {"name": "distill wide", "op": "distill", "r": 2048, "v": 131072, "top": 128, "type": "bf16", "step": False},
    ]


def _spread(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    op = rng.choice(["linear", "adjust", "draw", "distill"])
    kind = rng.choice(["f32", "bf16", "f16"])
    if op == "linear":
        k, n = _spread(rng, 16, 16384), _spread(rng, 16, 65536)
        return {"op": op, "m": _spread(rng, 1, min(16384, max(1, (1 << 38) // (k * n)))), "k": k, "n": n, "type": kind, "bias": rng.random() < 0.5}
    if op == "adjust":
        v = _spread(rng, 32, 262144)
        return {"op": op, "r": _spread(rng, 1, min(512, (1 << 24) // v)), "v": v, "type": kind, "history": _spread(rng, 1, 16384), "biases": rng.choice([0, 7, 100]),
                "masks": rng.choice([0, 1, 5])}
    if op == "draw":
        v = _spread(rng, 2, 262144)
        return {"op": op, "r": _spread(rng, 1, min(4096, (1 << 24) // v)), "v": v, "type": kind, "noise": rng.random() < 0.5}
    v = _spread(rng, 32, 262144)
    return {"op": op, "r": _spread(rng, 1, min(8192, (1 << 26) // v)), "v": v, "top": min(v, _spread(rng, 1, 256)), "type": kind, "step": rng.random() < 0.5}


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(int(seed) * 2 + 1)
    dt = TYPES[case["type"]]

    def normal(*size):
        return torch.randn(*size, generator=g, device="cuda")

    def uniform(*size):
        return torch.rand(*size, generator=g, device="cuda")

    def whole(low, high, *size, dtype=torch.int64):
        return torch.randint(low, high, size, generator=g, device="cuda", dtype=dtype)

    s = dict(case)
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        # activations with some channels an order of magnitude above the others; rows start on 16-byte boundaries, as weights that are laid out once do
        s["x"] = (normal(m, k) * torch.where(uniform(k) < 0.02, 12.0, 1.0)).to(dt)
        s["w"] = whole(-127, 128, n, (k + 15) // 16 * 16, dtype=torch.int8)[:, :k]
        s["w_scale"] = (0.5 + uniform(n)) * (0.02 / 127)
        s["b"] = normal(n) * 0.1 if case["bias"] else None
        return s
    if case["op"] == "draw":
        r, v = case["r"], case["v"]
        s["logits"] = (normal(r, v) * 3).masked_fill_(uniform(r, v) < 0.25, -math.inf).to(dt)
        s["beta"] = 0.5 + uniform(r)
        s["beta"][::5] = math.inf  # every fifth row is greedy
        s["u"] = ((whole(0, 1 << 23, r, v).float() + 0.5) * 2.0**-23) if case["noise"] else None
        s["key"] = int(whole(0, 1 << 62, 1).item())
        return s
    if case["op"] == "adjust":
        r, v = case["r"], case["v"]
        s["logits"] = (normal(r, v) * 3).to(dt)
        lengths = whole(case["history"] // 2, case["history"] + 1, r)
        s["ptr"] = torch.cat([lengths.new_zeros(1), lengths.cumsum(0)])
        # tokens come back: small ids far more often than large ones
        s["tokens"] = (uniform(int(s["ptr"][-1])).pow(3) * v).long().clamp_(max=v - 1).int()
        s["n_prompt"] = (lengths * uniform(r)).int()
        s["repetition"], s["frequency"], s["presence"] = 1 + 0.3 * uniform(r), 0.4 * uniform(r), 0.5 * uniform(r)
        s["bias_ids"] = s["bias_values"] = s["bias_ptr"] = s["mask"] = s["mask_rows"] = None
        if case["biases"]:
            s["bias_ids"] = whole(0, v, r, case["biases"], dtype=torch.int32).sort(1)[0].reshape(-1)
            s["bias_values"] = normal(r * case["biases"])
            s["bias_ptr"] = torch.arange(r + 1, device="cuda") * case["biases"]
        if case["masks"]:
            s["mask"] = whole(-(1 << 31), 1 << 31, case["masks"], (v + 31) // 32, dtype=torch.int32)
            s["mask_rows"] = whole(-1, case["masks"], r, dtype=torch.int32)  # -1: the row has no mask
        return s
    r, v, top = case["r"], case["v"], case["top"]
    s["logits"] = (normal(r, v) * 3).to(dt)
    s["ids"] = (uniform(r, 1) * v).int() + torch.arange(top, device="cuda", dtype=torch.int32) * max(1, v // top)
    s["ids"] = s["ids"].remainder(v)
    s["ids"][uniform(r, top) < 0.05] = -1  # fewer listed than `top`
    s["teacher"] = (normal(r, top) * 2).to(dt)
    s["weight"] = (uniform(r) > 0.1).float() / r  # a tenth of the rows is padding
    s["beta"] = 0.5
    return s


def run(state):
    return {"linear": _linear, "adjust": _adjust, "draw": _draw, "distill": _distill}[state["op"]](state)


def _framework():
    import __graft_entry__

    return __graft_entry__.load_package()


def _linear(s):
    if own:
        return _framework().int8_linear(s["x"], s["w"], s["w_scale"], s["b"])
    x = s["x"].float()
    scale = x.abs().amax(1, keepdim=True) / 127
    q = (x.double() / scale.double()).nan_to_num(0.0).round().clamp(-127, 127).float()  # in 64 bits: halves are borders
    y = (q @ s["w"].float().T) * scale * s["w_scale"]
    return (y if s["b"] is None else y + s["b"]).to(s["x"].dtype)


def _adjust(s):
    if own:
        return _framework().adjust_logits(s["logits"], history=s["tokens"], history_ptr=s["ptr"], n_prompt=s["n_prompt"], repetition=s["repetition"], frequency=s["frequency"],
                                          presence=s["presence"], bias_ids=s["bias_ids"], bias_values=s["bias_values"], bias_ptr=s["bias_ptr"], mask=s["mask"],
                                          mask_rows=s["mask_rows"])
    x = s["logits"].float()
    r, v = x.shape
    total = s["tokens"].numel()
    row = torch.repeat_interleave(torch.arange(r, device=x.device), s["ptr"].diff(), output_size=total)
    at = row * v + s["tokens"]
    seen = torch.zeros(r * v, device=x.device).index_add_(0, at, torch.ones(total, device=x.device)).view(r, v)
    behind = (torch.arange(total, device=x.device) - s["ptr"][row] >= s["n_prompt"][row]).float()
    told = torch.zeros(r * v, device=x.device).index_add_(0, at, behind).view(r, v)
    rep = s["repetition"][:, None]
    x = torch.where(seen > 0, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["frequency"][:, None] * told - s["presence"][:, None] * (told > 0)
    if s["bias_ids"] is not None:
        row = torch.repeat_interleave(torch.arange(r, device=x.device), s["bias_ptr"].diff(), output_size=s["bias_ids"].numel())
        x = x.reshape(-1).index_add(0, row * v + s["bias_ids"], s["bias_values"]).view(r, v)
    if s["mask"] is not None:
        k = torch.arange(v, device=x.device)
        open_ = (s["mask"][s["mask_rows"].clamp(min=0).long()][:, k >> 5] >> (k & 31)) & 1
        x = torch.where((open_ == 0) & (s["mask_rows"] >= 0)[:, None], -math.inf, x)
    return x.to(s["logits"].dtype)


def _round(c, k0, k1):
    """One round of Philox4x32 on 32-bit words held in int64."""
    low = 0xFFFFFFFF
    p, q = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57  # products modulo 2^64; the shifted half is masked, so the sign does not matter
    return ((q >> 32) & low) ^ c[1] ^ k0, q & low, ((p >> 32) & low) ^ c[3] ^ k1, p & low


def _uniforms(key, r, v, device):
    """Word k & 3 of Philox4x32-10(counter (row, 0, k >> 2, tag), key) as a 23-bit uniform inside (0, 1)."""
    row = torch.arange(r, device=device)[:, None].expand(r, (v + 3) // 4)
    zero = torch.zeros_like(row)
    c = (row, zero, torch.arange((v + 3) // 4, device=device).expand_as(row), zero + TAG_DRAW)
    for i in range(10):
        c = _round(c, ((key & 0xFFFFFFFF) + i * 0x9E3779B9) & 0xFFFFFFFF, ((key >> 32) + i * 0xBB67AE85) & 0xFFFFFFFF)
    words = torch.stack(c, 2).view(r, -1)[:, :v]
    return ((words >> 9).float() + 0.5) * 2.0**-23


def _draw(s):
    if own:
        return _framework().draw_categories(s["logits"], s["key"], beta=s["beta"], noise=s["u"])
    l = s["logits"].double()  # in 64 bits: two scores may lie next to each other
    u = _uniforms(s["key"], *l.shape, l.device) if s["u"] is None else s["u"]
    beta = s["beta"].double()[:, None]
    score = torch.where(beta.isinf(), l, torch.where(beta.isinf(), 0.0, beta) * l - (-u.double().log()).log())
    best = score.amax(1, keepdim=True)
    k = torch.arange(l.shape[1], device=l.device)
    first = torch.where(score == best, k, l.shape[1]).amin(1)
    return torch.where(best[:, 0] == -math.inf, -1, first)


def _distill(s):
    if own:
        T = _framework()
        if s["step"]:
            return T.distill_step(s["logits"], s["ids"], s["teacher"], beta=s["beta"], weight=s["weight"])
        loss, lse = T.distill_loss(s["logits"], s["ids"], s["teacher"], beta=s["beta"], weight=s["weight"])
        return loss, T.distill_grad(s["logits"], lse, s["ids"], s["teacher"], beta=s["beta"], weight=s["weight"])
    z, beta, live = s["logits"].float(), s["beta"], s["weight"] != 0
    z = z * beta
    top = z.amax(1, keepdim=True)
    e = (z - top).exp()
    total = e.sum(1, keepdim=True)
    there = s["ids"] >= 0
    at = s["ids"].clamp(min=0).long()
    t = torch.where(there, s["teacher"].float() * beta, -math.inf)
    t = t - t.amax(1, keepdim=True)
    t = torch.where(there, t - t.exp().sum(1, keepdim=True).log(), -math.inf)
    p = t.exp()
    term = torch.where(p > 0, p * (t - (z.gather(1, at) - top - total.log())), 0.0)
    some = there.any(1) & live  # a row without a teacher, or of weight 0, has no loss and no gradient
    loss = torch.where(some, term.sum(1), 0.0)
    grad = (e / total).scatter_add_(1, at, -torch.where(there, p, 0.0)) * (s["weight"] * beta)[:, None]
    return loss, torch.where(some[:, None], grad, 0.0).to(s["logits"].dtype)


def work(case):
    size = SIZE[case["type"]]
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        return {"bytes": m * k * size + n * k + 4 * n + m * n * size + (4 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    r, v = case["r"], case["v"]
    if case["op"] == "adjust":  # logits in and out, three quarters of `history` tokens a row, the biases, the masks
        return {"bytes": 2 * r * v * size + r * (3 * case["history"] + 8 * case["biases"] + 40) + case["masks"] * v / 8, "flops": 2 * r * v}
    if case["op"] == "draw":  # logits (and uniforms) in; a scale, a sum, two logarithms and a comparison for each
        return {"bytes": r * v * (size + (4 if case["noise"] else 0)) + 12 * r, "flops": 5 * r * v}
    # one pass: logits in, gradient out; two calls: logits in once more
    return {"bytes": (2 if case["step"] else 3) * r * v * size + r * case["top"] * (4 + size) * (1 if case["step"] else 2) + 12 * r, "flops": 6 * r * v}


def exact(case, seed):
    if case["op"] == "draw":  # category indices: no computed numbers
        return None
    s = prepare(case, seed)
    if case["op"] == "linear":
        x = s["x"].double()
        scale = (s["x"].float().abs().max(1).values / 127).double()  # the scale itself is held in 32 bits
        q = torch.nan_to_num(x / scale[:, None], nan=0.0).round().clamp(-127, 127)
        y = torch.einsum("mk,nk->mn", q, s["w"].double()) * torch.outer(scale, s["w_scale"].double())
        return y if s["b"] is None else y + s["b"].double()
    if case["op"] == "adjust":
        rows = []
        v = case["v"]
        bit = torch.arange(32, device="cuda")
        ptr, n_prompt = s["ptr"].tolist(), s["n_prompt"].tolist()
        for i in range(case["r"]):
            x = s["logits"][i].double()
            tokens = s["tokens"][ptr[i]:ptr[i + 1]].long()
            every, behind = torch.bincount(tokens, minlength=v), torch.bincount(tokens[n_prompt[i]:], minlength=v)
            rep = s["repetition"][i].double()
            x = torch.where(every > 0, x * rep ** (-x.sign()), x)
            x -= s["frequency"][i].double() * behind + s["presence"][i].double() * behind.clamp(max=1)
            if s["bias_ids"] is not None:
                mine = slice(i * case["biases"], (i + 1) * case["biases"])
                x += torch.bincount(s["bias_ids"][mine].long(), s["bias_values"][mine].double(), minlength=v)
            if s["mask"] is not None and s["mask_rows"][i] >= 0:
                allowed = (s["mask"][s["mask_rows"][i]][:, None] >> bit) & 1
                x[allowed.reshape(-1)[:v] == 0] = -math.inf
            rows.append(x)
        return torch.stack(rows)
    z = s["logits"].double() * s["beta"]
    log_q = z.log_softmax(1)
    there = s["ids"] >= 0
    t = (s["teacher"].double() * s["beta"]).masked_fill(~there, -math.inf)
    log_p = t.log_softmax(1)
    log_p[~there.any(1)] = -math.inf
    p = log_p.exp()
    at = s["ids"].clamp(min=0).long()
    loss = torch.where(p > 0, p * (log_p - log_q.gather(1, at)), 0).sum(1)
    grad = log_q.exp_().scatter_add_(1, at, -p).mul_((s["weight"].double() * s["beta"])[:, None])
    dead = ~there.any(1) | (s["weight"] == 0)
    loss[dead] = 0
    grad[dead] = 0
    return loss, grad
