"""The operators of a mixture of experts as cases that can be timed and checked: the router, the experts' products over
ragged groups of rows, the 8-bit products with a scale for each block of 128, and the weighted sum over a token's experts.

``own`` chooses the side: the plain form in elementary torch operations, or the calls a user makes of
``kudnn_amd.torch_moe``. ``listed`` has the calls that stand for the use of each operator, ``draw`` gives others of the
same ranges. Sizes are the benchmark's layer widths and generic transformer widths.
"""
import math

import torch

own = False

_TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_F8 = torch.float8_e4m3fn
_F8_MAX = 448.0          # largest e4m3 value: what a block's largest magnitude is scaled to
_TINY = 2.0 ** -126      # least scale of a block, the smallest normal f32


# ---- cases ------------------------------------------------------------------------------------------------------

def _route(tokens, experts, k, dtype, normalize=True, masked=False, train=False):
    return {"op": "route", "tokens": tokens, "experts": experts, "k": k, "dtype": dtype, "normalize": normalize,
            "masked": masked, "train": train}


def _grouped(tokens, experts, k, width, out, dtype, gather=True, train=False):
    return {"op": "grouped", "tokens": tokens, "experts": experts, "k": k, "width": width, "out": out, "dtype": dtype,
            "gather": gather, "train": train}


def _fp8(tokens, width, out, dtype, bias=False, experts=0, k=0):
    return {"op": "fp8", "tokens": tokens, "width": width, "out": out, "dtype": dtype, "bias": bias, "experts": experts,
            "k": k}


def _combine(tokens, experts, k, width, dtype, train=False):
    return {"op": "combine", "tokens": tokens, "experts": experts, "k": k, "width": width, "dtype": dtype, "train": train}


def listed():
    return [
        # The router of one decoded token, 8 of 64 experts: the smallest call, all launch and host.
        dict(_route(1, 64, 8, "bf16"), name="route_token"),
        # The router of a long batch of prompts, 8 of 128 experts: the sort by expert counts.
        dict(_route(16384, 128, 8, "bf16"), name="route_prefill"),
        # A training step's router in f32 over an odd number of tokens, some of them padding and some experts closed,
        # weights of the whole softmax, with the gradient of the logits.
        dict(_route(5003, 60, 4, "f32", normalize=False, masked=True, train=True), name="route_train"),
        # One token through its 8 experts' first product: 8 weights are streamed, a row for each.
        dict(_grouped(1, 64, 8, 2048, 4096, "bf16"), name="experts_token"),
        # A prompt through the second product of 32 experts, rows already in the experts' order, an odd output width.
        dict(_grouped(4096, 32, 4, 2048, 2824, "f16", gather=False), name="experts_prefill"),
        # A training step of 8 wide experts, 2 a token: product, gradient of the tokens, gradient of the weights.
        dict(_grouped(8192, 8, 2, 4096, 4096, "bf16", train=True), name="experts_train"),
        # The same for many small experts with an odd token count.
        dict(_grouped(3001, 48, 4, 1024, 1280, "bf16", train=True), name="experts_train_small"),
        # One token through the MLP's gate (C4's width) kept in 8 bits: the weight is streamed.
        dict(_fp8(1, 4096, 14336, "bf16"), name="fp8_token"),
        # Prefill up the MLP (C3's sizes) in 8 bits, with a bias.
        dict(_fp8(4096, 4096, 11008, "bf16", bias=True), name="fp8_prefill"),
        # A decode batch through 64 experts kept in 8 bits: some 64 ragged rows an expert.
        dict(_fp8(512, 2048, 4096, "bf16", experts=64, k=8), name="fp8_experts"),
        # The sum over 8 experts of a small decode batch.
        dict(_combine(16, 64, 8, 4096, "bf16"), name="combine_decode"),
        # A training step's sum with the gradients of the experts' rows and of the weights.
        dict(_combine(8192, 32, 4, 4096, "bf16", train=True), name="combine_train"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A layer's width: usually a multiple of 128 or 64, at times only of 8, seldom odd."""
    step = rng.choice((128, 128, 128, 64, 64, 8, 8, 1))
    v = max(lo, min(hi, int(round(_log(rng, lo, hi) / step)) * step))
    return v + 128 if v == 3072 else v


def _drawn(rng):
    op = rng.choice(["route", "grouped", "grouped", "grouped", "fp8", "fp8", "combine"])
    experts = rng.choice([8, 16, 32, 60, 64, 128])
    k = rng.randint(1, min(8, experts))
    half = rng.choice(["bf16", "bf16", "f16"])
    if op == "route":
        experts = rng.choice([experts, _log(rng, 4, 256)])
        return _route(_log(rng, 1, 16384), experts, min(k, experts), rng.choice(["bf16", "f32", "f16"]),
                      rng.random() < 0.5, rng.random() < 0.4, rng.random() < 0.4)
    if op == "combine":
        return _combine(_log(rng, 1, 8192), experts, k, _width(rng, 256, 4096), rng.choice(["bf16", "f16", "f32"]),
                        rng.random() < 0.5)
    width, out = _width(rng, 256, 8192), _width(rng, 256, 8192)
    if op == "fp8" and rng.random() < 0.5:
        return _fp8(_log(rng, 1, 4096), width, out, half, rng.random() < 0.5)
    if op == "fp8":
        return _fp8(_log(rng, 1, 4096), width, out, half, False, experts, k)
    train = rng.random() < 0.4
    return _grouped(_log(rng, 64 if train else 1, 8192), experts, k, width, out, half, rng.random() < 0.6, train)


def draw(rng):
    """A case of the listed ones' ranges that has no more to move or to compute than the largest of its operator."""
    while True:
        c = _drawn(rng)
        mine, largest = work(c), [work(x) for x in listed() if x["op"] == c["op"]]
        if all(mine[n] <= max(x[n] for x in largest) for n in mine):
            return c


def work(case):
    t, e, k = case["tokens"], case["experts"], case["k"]
    if case["op"] == "route":
        size = 4 if case["dtype"] == "f32" else 2
        n = t * e * size + (t * e if case["masked"] else 0) + t * k * 4 * 4 + (e + 1) * 4
        return {"bytes": n + (t * k * 4 + t * e * size if case["train"] else 0), "flops": 4 * t * e * (2 if case["train"] else 1)}
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "combine":
        d = case["width"]
        n = (t * k * d + t * d) * size + t * k * 8
        return {"bytes": 2 * n + t * k * d * size if case["train"] else n, "flops": 2 * t * k * d * (3 if case["train"] else 1)}
    kd, n = case["width"], case["out"]
    if case["op"] == "fp8":
        rows = t * k if e else t
        weights = min(e, rows) if e else 1
        blocks = ((n + 127) // 128) * ((kd + 127) // 128)
        return {"bytes": t * kd * size + weights * (n * kd + 4 * blocks) + rows * n * size + (n * size if case["bias"] else 0),
                "flops": 2 * rows * kd * n}
    rows, weights = t * k, min(e, t * k)
    x = (t if case["gather"] else rows) * kd
    one = x + weights * kd * n + rows * n
    return {"bytes": one * size + (one + rows * n) * size if case["train"] else one * size,
            "flops": 2 * rows * kd * n * (3 if case["train"] else 1)}


# ---- inputs -----------------------------------------------------------------------------------------------------

def _quantize_weight(w):
    """[..., N, K] -> e4m3 values and the f32 scale of each block of 128 x 128."""
    n, k = w.shape[-2:]
    nb, kb = (n + 127) // 128, (k + 127) // 128
    full = torch.nn.functional.pad(w, (0, kb * 128 - k, 0, nb * 128 - n))
    blocks = full.reshape(*w.shape[:-2], nb, 128, kb, 128)
    scale = torch.clamp(blocks.abs().amax((-3, -1)) / _F8_MAX, min=_TINY)
    q = (blocks / scale[..., :, None, :, None]).reshape(full.shape)[..., :n, :k]
    return q.contiguous().to(_F8), scale


def _plan_of(experts, count):
    """Chosen experts [T, k] (-1: none) -> offsets [E + 1], rows [T k] and slots [T, k] of the order by expert."""
    t, k = experts.shape
    key = torch.where(experts < 0, count, experts).reshape(-1).long()
    order = torch.sort(key, stable=True).indices
    sorted_key = key[order]
    offsets = (sorted_key[:, None] < torch.arange(count + 1, device=key.device)[None, :]).sum(0)
    chosen = sorted_key < count
    rows = torch.where(chosen, order // k, -1)
    slots = torch.empty_like(order)
    slots[order] = torch.where(chosen, torch.arange(t * k, device=key.device), -1)
    return offsets.int(), rows.int(), slots.reshape(t, k).int()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)

    t, e, k, op = case["tokens"], case["experts"], case["k"], case["op"]
    dt = _TORCH[case["dtype"]]
    s = {"case": case}
    if op == "fp8" and not e:
        s["x"] = (randn(t, case["width"]) * torch.exp(randn(1, case["width"]))).to(dt)
        s["w"], s["ws"] = _quantize_weight(randn(case["out"], case["width"]) * case["width"] ** -0.5)
        s["bias"] = (randn(case["out"]) * 0.1).to(dt) if case["bias"] else None
        return s
    # a router's scores: tokens differ, and some experts are liked by most
    logits = randn(t, e) * 1.5 + randn(1, e) * 0.5
    if op == "route":
        s["logits"] = logits.to(dt)
        s["mask"] = None
        if case["masked"]:
            # every 16th token is padding, and a token may not go to an eighth of the experts
            mask = torch.rand(t, e, generator=g, device="cuda") >= 0.125
            mask[::16] = False
            s["mask"] = mask
        if case["train"]:
            s["logits"].requires_grad_(True)
            s["dweights"] = randn(t, k)
        return s
    experts = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :k].int()
    s["offsets"], s["rows"], s["slots"] = _plan_of(experts, e)
    if op == "combine":
        s["y"] = randn(t * k, case["width"]).to(dt)
        s["weights"] = torch.softmax(randn(t, k), 1)
        if case["train"]:
            s["y"].requires_grad_(True)
            s["weights"].requires_grad_(True)
            s["dout"] = randn(t, case["width"]).to(dt)
        return s
    kd, n = case["width"], case["out"]
    s["most"] = int((s["offsets"][1:] - s["offsets"][:-1]).max())  # rows of the fullest expert, for the plain form
    if op == "fp8":
        s["x"] = (randn(t, kd) * torch.exp(randn(1, kd))).to(dt)
        w = torch.empty(e, n, kd, device="cuda", dtype=_F8)
        ws = torch.empty(e, (n + 127) // 128, (kd + 127) // 128, device="cuda", dtype=torch.float32)
        for i in range(e):
            w[i], ws[i] = _quantize_weight(randn(n, kd) * kd ** -0.5)
        s["w"], s["ws"] = w, ws
        return s
    s["x"] = randn(t if case["gather"] else t * k, kd).to(dt)
    w = torch.empty(e, n, kd, device="cuda", dtype=dt)
    for i in range(e):
        w[i] = randn(n, kd) * kd ** -0.5
    s["w"] = w
    if case["train"]:
        s["x"].requires_grad_(True)
        s["w"].requires_grad_(True)
        s["dy"] = randn(t * k, n).to(dt)
    return s


# ---- the plain forms --------------------------------------------------------------------------------------------

def _plain_route(s, c):
    # p = softmax of the open experts' logits; the k largest, ties to the lowest index; weights p, or p over their sum
    logits = s["logits"].detach().float()
    t, e = logits.shape
    k = c["k"]
    open_ = torch.isinf(logits).logical_not() | (logits > 0)
    if s["mask"] is not None:
        open_ = open_ & s["mask"]
    lowest = torch.full_like(logits, -math.inf)
    x = torch.where(open_, logits, lowest)
    top = x.amax(1, keepdim=True)
    p = torch.where(open_, torch.exp(x - torch.where(torch.isinf(top), 0.0, top)), 0.0)
    total = p.sum(1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k]
    some = open_.gather(1, order)
    experts = torch.where(some, order, -1).int()
    picked = torch.where(some, p.gather(1, order), 0.0)
    whole = picked.sum(1, keepdim=True)
    weights = picked / torch.where(whole == 0, 1.0, whole) if c["normalize"] else picked
    offsets, rows, slots = _plan_of(experts, e)
    outs = [weights, experts, offsets, rows, slots]
    if c["train"]:
        gw = torch.where(some, s["dweights"], 0.0)
        dot = (gw * weights).sum(1, keepdim=True)
        dx = torch.zeros_like(logits)
        if c["normalize"]:
            dx.scatter_add_(1, order, torch.where(some, weights * (gw - dot), 0.0))
        else:
            dx.scatter_add_(1, order, weights * gw)
            dx -= p * dot
        outs.append(dx.to(s["logits"].dtype))
    return outs


def _groups(s):
    """The expert of each row and the row's place in its group."""
    r = torch.arange(s["rows"].shape[0], device="cuda")
    expert = (r[:, None] >= s["offsets"][None, 1:]).sum(1)
    return expert, r - s["offsets"].long()[expert]


def _padded(x, s, expert, place):
    full = torch.zeros(s["offsets"].shape[0] - 1, s["most"], x.shape[1], device="cuda", dtype=torch.float32)
    full[expert, place] = x
    return full


def _plain_product(s, c, x, weight):
    """Rows in the experts' order times their expert's weight [N, K], in f32; weight(index) gives the weights in f32."""
    expert, place = _groups(s)
    if x.shape[0] <= s["w"].shape[0]:
        # fewer rows than experts: a weight for each row
        return (weight(expert) * x[:, None, :]).sum(2)
    return torch.bmm(_padded(x, s, expert, place), weight(slice(None)).transpose(1, 2).contiguous())[expert, place]


def _plain_grouped(s, c):
    x = s["x"].detach().float()
    w = s["w"].detach()
    xs = x[s["rows"].long()] if c["gather"] else x
    y = _plain_product(s, c, xs, lambda i: w[i].float())
    if not c["train"]:
        return y.to(w.dtype)
    expert, place = _groups(s)
    dy = _padded(s["dy"].float(), s, expert, place)
    dx = torch.bmm(dy, w.float())[expert, place]
    if c["gather"]:
        dx = dx[s["slots"].long()].sum(1)
    dw = torch.bmm(dy.transpose(1, 2).contiguous(), _padded(xs, s, expert, place))
    return [y.to(w.dtype), dx.to(w.dtype), dw.to(w.dtype)]


def _plain_fp8(s, c):
    x = s["x"].float()
    m, kd = x.shape
    n, kb = c["out"], (kd + 127) // 128
    # a scale for each row's block of 128: its largest magnitude over 448; the values rounded to e4m3
    blocks = torch.nn.functional.pad(x, (0, kb * 128 - kd)).reshape(m, kb, 128)
    scale = torch.clamp(blocks.abs().amax(2) / _F8_MAX, min=_TINY)
    xq = ((blocks / scale[:, :, None]).to(_F8).float() * scale[:, :, None]).reshape(m, kb * 128)[:, :kd]

    def weight(i):
        ws = s["ws"][i] if c["experts"] else s["ws"]
        full = ws.repeat_interleave(128, -2)[..., :n, :].repeat_interleave(128, -1)[..., :kd]
        return (s["w"][i] if c["experts"] else s["w"]).float() * full

    if c["experts"]:
        return _plain_product(s, c, xq[s["rows"].long()], weight).to(s["x"].dtype)
    y = xq @ weight(None).t()
    return (y if s["bias"] is None else y + s["bias"].float()).to(s["x"].dtype)


def _plain_combine(s, c):
    y, w, slots = s["y"].detach().float(), s["weights"].detach(), s["slots"].long()
    picked = y[slots]
    out = (picked * w[:, :, None]).sum(1).to(s["y"].dtype)
    if not c["train"]:
        return out
    dout = s["dout"].float()
    dw = (picked * dout[:, None, :]).sum(2)
    dy = torch.zeros_like(y)
    dy[slots.reshape(-1)] = (w[:, :, None] * dout[:, None, :]).reshape(-1, y.shape[1])
    return [out, dy.to(s["y"].dtype), dw]


# ---- the framework's calls --------------------------------------------------------------------------------------

def _own(s, c):
    import kudnn_amd.torch_moe as km

    op = c["op"]
    if op == "route":
        r = km.route(s["logits"], c["k"], normalize=c["normalize"], mask=s["mask"])
        outs = [r.weights.detach(), r.experts, r.offsets, r.rows, r.slots]
        if c["train"]:
            outs += torch.autograd.grad(r.weights, s["logits"], s["dweights"])
        return outs
    if op == "grouped":
        rows = s["rows"] if c["gather"] else None
        if not c["train"]:
            return km.grouped_linear(s["x"], s["w"], s["offsets"], rows)
        y = km.grouped_linear(s["x"], s["w"], s["offsets"], rows, s["slots"] if c["gather"] else None)
        return [y.detach(), *torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])]
    if op == "fp8":
        if c["experts"]:
            return km.grouped_linear_fp8(s["x"], s["w"], s["ws"], s["offsets"], s["rows"])
        return km.linear_fp8(s["x"], s["w"], s["ws"], s["bias"])
    if not c["train"]:
        return km.combine(s["y"], s["weights"], s["slots"])
    out = km.combine(s["y"], s["weights"], s["slots"])
    return [out.detach(), *torch.autograd.grad(out, (s["y"], s["weights"]), s["dout"])]


_PLAIN = {"route": _plain_route, "grouped": _plain_grouped, "fp8": _plain_fp8, "combine": _plain_combine}


def run(state):
    case = state["case"]
    return _own(state, case) if own else _PLAIN[case["op"]](state, case)


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------

def _exact_route(s, c):
    x = s["logits"].detach().cpu().double()
    t, e = x.shape
    open_ = x != -math.inf
    if s["mask"] is not None:
        open_ &= s["mask"].cpu()
    out = torch.zeros(t, c["k"], dtype=torch.float64)
    grads = torch.zeros(t, e, dtype=torch.float64)
    # the whole softmax, the chosen of it, and the Jacobian's product with the gradient of the chosen weights
    soft = torch.nan_to_num(torch.softmax(x.masked_fill(~open_, -math.inf), 1), nan=0.0)
    ranked = torch.sort(x.masked_fill(~open_, -math.inf), dim=1, descending=True, stable=True).indices[:, :c["k"]]
    mine = soft.gather(1, ranked) * open_.gather(1, ranked)
    if c["normalize"]:
        out = mine / mine.sum(1, keepdim=True).clamp_min(1e-300)
    else:
        out = mine
    if c["train"]:
        gw = s["dweights"].cpu().double()
        mean = (gw * out).sum(1, keepdim=True)
        share = torch.zeros(t, e, dtype=torch.float64).scatter_(1, ranked, gw * open_.gather(1, ranked))
        hit = torch.zeros(t, e, dtype=torch.float64).scatter_(1, ranked, open_.gather(1, ranked).double())
        grads = (hit * soft / (hit * soft).sum(1, keepdim=True).clamp_min(1e-300) * (share - mean)) if c["normalize"] \
            else soft * (share - mean)
    return [out, None, None, None, None] + ([grads] if c["train"] else [])


def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["op"] == "route":
        return _exact_route(s, c)
    if c["op"] == "combine":
        y, w = s["y"].detach().double(), s["weights"].detach().double()
        t, k = w.shape
        out = torch.zeros(t, c["width"], device="cuda", dtype=torch.float64)
        dy, dw = torch.zeros_like(y), torch.zeros_like(w)
        for j in range(k):
            at = s["slots"][:, j].long()
            out += w[:, j:j + 1] * y[at]
            if c["train"]:
                dout = s["dout"].double()
                dy[at] = w[:, j:j + 1] * dout
                dw[:, j] = (dout * y[at]).sum(1)
        return [out, dy, dw] if c["train"] else out
    kd, n = c["width"], c["out"]
    if c["op"] == "fp8":
        x = s["x"].float()
        xq = torch.empty(x.shape, device="cuda", dtype=torch.float64)
        for b in range(0, kd, 128):
            part = x[:, b:b + 128]
            scale = (part.abs().max(1, keepdim=True).values / _F8_MAX).clamp_min(_TINY)
            xq[:, b:b + 128] = (part / scale).to(_F8).double() * scale.double()

        def weight(w, ws):
            w = w.double()
            for i in range(ws.shape[0]):
                for j in range(ws.shape[1]):
                    w[i * 128:i * 128 + 128, j * 128:j * 128 + 128] *= ws[i, j].double()
            return w

        if not c["experts"]:
            y = xq @ weight(s["w"], s["ws"]).t()
            return y if s["bias"] is None else y + s["bias"].double()
        xs = xq[s["rows"].long()]
        offsets = s["offsets"].tolist()
        y = torch.zeros(xs.shape[0], n, device="cuda", dtype=torch.float64)
        for i, (lo, hi) in enumerate(zip(offsets, offsets[1:])):
            if hi > lo:
                y[lo:hi] = xs[lo:hi] @ weight(s["w"][i], s["ws"][i]).t()
        return y
    xs = s["x"].detach()
    xs = xs[s["rows"].long()] if c["gather"] else xs
    offsets = s["offsets"].tolist()
    y = torch.zeros(xs.shape[0], n, device="cuda", dtype=torch.float64)
    dxs = torch.zeros(xs.shape[0], kd, device="cuda", dtype=torch.float64) if c["train"] else None
    dw = torch.zeros(c["experts"], n, kd, device="cuda", dtype=torch.float64) if c["train"] else None
    for i, (lo, hi) in enumerate(zip(offsets, offsets[1:])):
        if hi > lo:
            w = s["w"][i].detach().double()
            y[lo:hi] = xs[lo:hi].double() @ w.t()
            if c["train"]:
                dy = s["dy"][lo:hi].double()
                dxs[lo:hi] = dy @ w
                dw[i] = dy.t() @ xs[lo:hi].double()
    if not c["train"]:
        return y
    if c["gather"]:
        dx = torch.zeros(c["tokens"], kd, device="cuda", dtype=torch.float64)
        dx.index_add_(0, s["rows"].long(), dxs)
    else:
        dx = dxs
    return [y, dx, dw]
