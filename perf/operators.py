"""Cases, plain forms and 64-bit values of three groups of operators:

  layernorm   normalisation over the last (channel) dimension, with the
              gradients of input, gamma and beta
  logprobs    log probability of each row's given class, entropy and the
              top alternatives, with the gradient of the logits
  muon        the orthogonalised momentum update: Newton-Schulz products
              of one matrix, of a batch, and of a network's whole
              parameter set

``listed()`` and ``draw()`` give cases, ``prepare()`` their inputs,
``run()`` one pass, in plain torch operations or (``own``) through the
framework's entry points; ``exact()`` the same in 64 bits.
"""

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16,
          "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-5                         # layernorm's default
STEPS = 5                          # Newton-Schulz products' default
QUINTIC = (3.4445, -4.775, 2.0315)
NORM_EPS = 1e-7
MOMENTUM, RMS = 0.95, 0.2

# the weights of the 16-layer CIFAR wide residual network, as matrices
# of output channels by (taps x input channels)
WRN = ("16x27,64x144,64x576,64x16,64x576,64x576,"
       "128x576,128x1152,128x64,128x1152,128x1152,"
       "256x1152,256x2304,256x128,256x2304,256x2304,10x256")


def listed():
    return [
        # the features in front of a classifier at a training batch of
        # 128: little data, so that latency counts
        {"name": "ln_128x4096_bf16_train", "op": "layernorm", "rows": 128,
         "width": 4096, "pad": 0, "dtype": "bf16", "train": True},
        # pooled features of a small batch when a model answers
        {"name": "ln_32x1024_f16", "op": "layernorm", "rows": 32,
         "width": 1024, "pad": 0, "dtype": "f16", "train": False},
        # the largest: every pixel of a residual network's first stage
        # at batch 256 (256 x 56 x 56 pixels of 256 channels)
        {"name": "ln_802816x256_bf16_train", "op": "layernorm",
         "rows": 802816, "width": 256, "pad": 0, "dtype": "bf16",
         "train": True},
        # class scores in the physical padding to 16 channels, in 32
        # bits, an odd number of rows
        {"name": "ln_4099x1000_f32_train", "op": "layernorm",
         "rows": 4099, "width": 1000, "pad": 8, "dtype": "f32",
         "train": True},
        # a 1000-way classifier's batch, channel-padded to 1008, with
        # the five best classes
        {"name": "lp_128x1000_bf16_train", "op": "logprobs", "rows": 128,
         "width": 1000, "pad": 8, "top": 5, "dtype": "bf16",
         "train": True, "banned": 0.0},
        # one row over a large set of classes: a single answer
        {"name": "lp_1x131072_f32", "op": "logprobs", "rows": 1,
         "width": 131072, "pad": 0, "top": 8, "dtype": "f32",
         "train": False, "banned": 0.0},
        # a training batch over a large set of classes
        {"name": "lp_2048x131072_bf16_train", "op": "logprobs",
         "rows": 2048, "width": 131072, "pad": 0, "top": 8,
         "dtype": "bf16", "train": True, "banned": 0.0},
        # odd sizes, many alternatives, a twentieth of the classes
        # masked out
        {"name": "lp_333x32771_f16_train", "op": "logprobs", "rows": 333,
         "width": 32771, "pad": 0, "top": 20, "dtype": "f16",
         "train": True, "banned": 0.05},
        # one 3x3 convolution's weight
        {"name": "ns_64x576_f32", "op": "orthogonalize", "batch": 1,
         "rows": 64, "cols": 576, "dtype": "f32"},
        # the first fully connected layer behind 6 x 6 x 256 features
        {"name": "ns_4096x9216_f32", "op": "orthogonalize", "batch": 1,
         "rows": 4096, "cols": 9216, "dtype": "f32"},
        # a batch of tall matrices of odd sizes
        {"name": "ns_12x333x201_bf16", "op": "orthogonalize", "batch": 12,
         "rows": 333, "cols": 201, "dtype": "bf16"},
        # one update of a whole network
        {"name": "muon_wresnet", "op": "muon", "shapes": WRN},
    ]


def _between(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(
        rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("layernorm", "logprobs", "orthogonalize", "muon"))
    if op == "layernorm":
        width = _between(rng, 16, 16384)
        rows = _between(rng, 1, min(802816, 802816 * 256 // (2 * width)))
        return {"op": op, "rows": rows, "width": width,
                "pad": rng.choice((0, 0, -width % 16)),
                "dtype": rng.choice(("bf16", "bf16", "f16", "f32")),
                "train": rng.random() < 0.7}
    if op == "logprobs":
        width = _between(rng, 10, 200000)
        rows = _between(rng, 1, min(16384, 2048 * 131072 // (2 * width)))
        return {"op": op, "rows": rows, "width": width,
                "pad": rng.choice((0, 0, -width % 16)),
                "top": rng.randint(0, min(20, width)),
                "dtype": rng.choice(("bf16", "bf16", "f16", "f32")),
                "train": rng.random() < 0.6,
                "banned": rng.choice((0.0, 0.0, 0.1))}
    if op == "orthogonalize":
        rows, cols = _between(rng, 16, 4096), _between(rng, 16, 9216)
        if rng.random() < 0.5:
            rows, cols = cols, rows
        one = _ns_flops(rows, cols)
        most = min(48, int(_ns_flops(4096, 9216) // (2 * one)))
        return {"op": op, "batch": _between(rng, 1, max(1, most)),
                "rows": rows, "cols": cols,
                "dtype": rng.choice(("f32", "f32", "bf16"))}
    shapes = ["%dx%d" % (_between(rng, 10, 1024), _between(rng, 16, 4608))
              for _ in range(rng.randint(1, 20))]
    return {"op": op, "shapes": ",".join(shapes)}


def _shapes(case):
    return [tuple(int(n) for n in s.split("x"))
            for s in case["shapes"].split(",")]


def _ns_flops(rows, cols):
    """The products of the recurrence: the Gram matrix (symmetric, so
    half of it), its square (half of it) and the product with X."""
    m, n = min(rows, cols), max(rows, cols)
    return STEPS * (m * m * n + m * m * m + 2.0 * m * m * n)


def work(case):
    if case["op"] == "layernorm":
        n = float(case["rows"] * (case["width"] + case["pad"]))
        size = SIZES[case["dtype"]]
        # x in, y out; training: dy in, dx out besides
        return {"bytes": n * size * (4 if case["train"] else 2),
                "flops": n * (20 if case["train"] else 8)}
    if case["op"] == "logprobs":
        n = float(case["rows"] * (case["width"] + case["pad"]))
        size = SIZES[case["dtype"]]
        # logits in; training: their gradient out besides
        return {"bytes": n * size * (2 if case["train"] else 1),
                "flops": n * (12 if case["train"] else 6)}
    if case["op"] == "orthogonalize":
        n = float(case["batch"] * case["rows"] * case["cols"])
        return {"bytes": 2 * n * SIZES[case["dtype"]],
                "flops": case["batch"] * _ns_flops(case["rows"],
                                                   case["cols"])}
    n = float(sum(r * c for r, c in _shapes(case)))
    # weight, gradient and momentum in, weight, momentum and the bf16
    # copy out
    return {"bytes": n * (3 * 4 + 2 * 4 + 2),
            "flops": sum(_ns_flops(r, c) for r, c in _shapes(case))}


def _gradient(gen, batch, rows, cols):
    """Like a layer's momentum: few strong directions, of falling
    strength, over the noise of the batch in all directions."""
    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")
    rank = max(1, min(16, min(rows, cols) // 4))
    left = normal(batch, rows, rank) * torch.logspace(
        0, -1, rank, device="cuda")
    strong = torch.bmm(left, normal(batch, rank, cols))
    return 1e-3 * (strong + 0.5 * normal(batch, rows, cols))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    if case["op"] == "layernorm":
        rows, n, pad = case["rows"], case["width"], case["pad"]
        dt = DTYPES[case["dtype"]]
        x = (1.5 * normal(rows, n + pad) + 0.5 * normal(n + pad)).to(dt)
        s = {"case": case, "x": x, "gamma": 1 + 0.2 * normal(n + pad),
             "beta": 0.1 * normal(n + pad)}
        if pad:                       # padded channels hold zeros
            for t in (s["x"], s["gamma"], s["beta"]):
                t[..., n:] = 0
        if case["train"]:
            s["dy"] = (normal(rows, n + pad) / 64).to(dt)
            for k in ("x", "gamma", "beta"):
                s[k].requires_grad_(True)
        return s
    if case["op"] == "logprobs":
        rows, n, pad = case["rows"], case["width"], case["pad"]
        x = 2.5 * normal(rows, n + pad)
        x[:, n:] = 0
        labels = torch.randint(0, n, (rows,), generator=gen,
                               device="cuda")
        # a classifier that has learned something: the given class
        # stands out in most rows
        x[torch.arange(rows, device="cuda"), labels] += 6 * torch.rand(
            rows, generator=gen, device="cuda")
        if case["banned"]:
            ban = torch.rand(n + pad, generator=gen, device="cuda")
            ban = (ban < case["banned"]).expand(rows, -1).clone()
            ban[torch.arange(rows, device="cuda"), labels] = False
            ban[:, n:] = False
            x.masked_fill_(ban, float("-inf"))
        s = {"case": case, "x": x.to(DTYPES[case["dtype"]]),
             "labels": labels}
        if case["train"]:
            s["dlogp"] = normal(rows) / 16
            s["dentropy"] = normal(rows) / 64
            s["dtop"] = normal(rows, case["top"]) / 64
            s["x"].requires_grad_(True)
        return s
    if case["op"] == "orthogonalize":
        x = _gradient(gen, case["batch"], case["rows"], case["cols"])
        x = x.to(DTYPES[case["dtype"]])
        return {"case": case, "x": x[0] if case["batch"] == 1 else x}
    s = {"case": case, "w": [], "g": [], "v": [], "out": [], "scale": []}
    for r, c in _shapes(case):
        w = normal(r, c) * math.sqrt(2.0 / c)
        s["w"].append(w)
        s["g"].append(_gradient(gen, 1, r, c)[0])
        s["v"].append(-8 * _gradient(gen, 1, r, c)[0])
        s["out"].append(w.to(torch.bfloat16))
        s["scale"].append(RMS * math.sqrt(max(r, c)))
    return s


def _plain_layernorm(s):
    case, n = s["case"], s["case"]["width"]
    x = s["x"].detach()[:, :n].float()
    gamma = s["gamma"].detach()[:n]
    d = x - x.mean(dim=1, keepdim=True)
    rstd = torch.rsqrt((d * d).mean(dim=1, keepdim=True) + EPS)
    xhat = d * rstd
    out = [xhat * gamma + s["beta"].detach()[:n]]
    if case["train"]:
        dy = s["dy"][:, :n].float()
        g = dy * gamma
        out += [rstd * (g - g.mean(dim=1, keepdim=True)
                        - xhat * (g * xhat).mean(dim=1, keepdim=True)),
                (dy * xhat).sum(dim=0), dy.sum(dim=0)]
    if case["pad"]:
        out = [torch.nn.functional.pad(t, (0, case["pad"])) for t in out]
    out[:2] = [t.to(s["x"].dtype) for t in out[:2]]
    return out


def _plain_logprobs(s):
    case, n, k = s["case"], s["case"]["width"], s["case"]["top"]
    x = s["x"].detach()[:, :n].float()
    d = x - x.amax(dim=1, keepdim=True)
    e = torch.exp(d)
    total = e.sum(dim=1, keepdim=True)
    logp = d - torch.log(total)
    p = e / total
    plogp = p * torch.where(e > 0, logp, torch.zeros_like(logp))
    entropy = -plogp.sum(dim=1)
    given = logp.gather(1, s["labels"][:, None])[:, 0]
    out = [given, entropy]
    if k:
        # keys that order as the values do, and equal values by index
        bits = (x + 0.0).view(torch.int32)
        bits = torch.where(bits >= 0, bits, bits ^ 0x7fffffff).long()
        last = 2 ** 31 - 1
        keys = bits * 2 ** 32 + (last - torch.arange(n, device=x.device))
        best = last - (keys.topk(k, dim=1).values & 0xffffffff)
        out += [logp.gather(1, best), best]
    if case["train"]:
        sums = s["dlogp"] + s["dtop"].sum(dim=1)
        dx = -p * sums[:, None] - s["dentropy"][:, None] * (
            plogp + p * entropy[:, None])
        dx.scatter_add_(1, s["labels"][:, None], s["dlogp"][:, None])
        if k:
            dx.scatter_add_(1, best, s["dtop"])
        out.append(torch.nn.functional.pad(
            dx, (0, case["pad"])).to(s["x"].dtype))
    return out


def _plain_orthogonalize(x):
    y = x.float()
    tall = y.shape[-2] > y.shape[-1]
    if tall:
        y = y.transpose(-2, -1)
    y = y / (y.square().sum(dim=(-2, -1), keepdim=True).sqrt() + NORM_EPS)
    a, b, c = QUINTIC
    for _ in range(STEPS):
        gram = y @ y.transpose(-2, -1)
        y = a * y + (b * gram + c * (gram @ gram)) @ y
    return (y.transpose(-2, -1) if tall else y).to(x.dtype)


LR, DECAY = 0.02, 0.01


def _plain_muon(s):
    for w, g, v, out, scale in zip(s["w"], s["g"], s["v"], s["out"],
                                   s["scale"]):
        v.mul_(MOMENTUM).sub_(g)
        w.mul_(1 - LR * DECAY).add_(_plain_orthogonalize(v),
                                    alpha=LR * scale)
        out.copy_(w)
    return [s["w"], s["v"], s["out"]]


def run(s):
    op = s["case"]["op"]
    if own:
        from theanompi_amd.ops import functional as OF
        if op == "layernorm":
            n, pad = s["case"]["width"], s["case"]["pad"]
            leaves = (s["x"], s["gamma"], s["beta"])
            y = OF.layernorm(*leaves, eps=EPS,
                             n_features=n if pad else None)
            if not s["case"]["train"]:
                return [y]
            return [y.detach(), *torch.autograd.grad(y, leaves, s["dy"])]
        if op == "logprobs":
            k = s["case"]["top"]
            out = OF.label_logprobs(
                s["x"], s["labels"], n_classes=s["case"]["width"], top=k)
            got = [t.detach() for t in out[:4 if k else 2]]
            if s["case"]["train"]:
                grads = (s["dlogp"], s["dentropy"], s["dtop"])
                got += torch.autograd.grad(out[:3 if k else 2], s["x"],
                                           grads[:3 if k else 2])
            return got
        if op == "orthogonalize":
            return [OF.orthogonalize(s["x"])]
        many = len(s["w"])
        OF.muon_update(s["w"], s["g"], s["v"], s["out"], [LR] * many,
                       [DECAY] * many, MOMENTUM, s["scale"])
        return [s["w"], s["v"], s["out"]]
    with torch.no_grad():
        if op == "layernorm":
            return _plain_layernorm(s)
        if op == "logprobs":
            return _plain_logprobs(s)
        if op == "orthogonalize":
            return [_plain_orthogonalize(s["x"])]
        return _plain_muon(s)


def _exact_orthogonal(x):
    """The recurrence in 64 bits, from the right: X <- X (a + bG + cG^2)
    with G = X^T X, on the orientation that has the fewer columns."""
    if x.shape[-2] < x.shape[-1]:
        return _exact_orthogonal(
            x.transpose(-2, -1).contiguous()).transpose(-2, -1)
    x = x / (torch.linalg.vector_norm(x, dim=(-2, -1), keepdim=True)
             + NORM_EPS)
    a, b, c = QUINTIC
    eye = torch.eye(x.shape[-1], dtype=x.dtype, device=x.device)
    for _ in range(STEPS):
        g = x.transpose(-2, -1).contiguous() @ x
        x = x @ (a * eye + g @ (b * eye + c * g))
    return x


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "layernorm":
        n, pad = case["width"], case["pad"]
        x, gamma, beta = (
            s[k].detach()[..., :n].double().requires_grad_(case["train"])
            for k in ("x", "gamma", "beta"))
        y = torch.nn.functional.layer_norm(x, (n,), gamma, beta, EPS)
        out = [y.detach()]
        if case["train"]:
            out += torch.autograd.grad(y, (x, gamma, beta),
                                       s["dy"][:, :n].double())
        return [torch.nn.functional.pad(t, (0, pad)) for t in out]
    if case["op"] == "logprobs":
        n, k = case["width"], case["top"]
        x = s["x"].detach()[:, :n].double().requires_grad_(case["train"])
        logp = torch.log_softmax(x, dim=1)
        finite = logp.masked_fill(x == float("-inf"), 0.0)
        entropy = -(logp.exp() * finite).sum(dim=1)
        out = [logp[torch.arange(len(x), device="cuda"), s["labels"]],
               entropy]
        if k:
            best = x.detach().sort(dim=1, descending=True,
                                   stable=True).indices[:, :k]
            out.append(logp.gather(1, best))
        got = [t.detach() for t in out] + ([best] if k else [])
        if case["train"]:
            grads = (s["dlogp"], s["dentropy"], s["dtop"])
            (dx,) = torch.autograd.grad(
                out, x, [g.double() for g in grads[:len(out)]])
            got.append(torch.nn.functional.pad(dx, (0, case["pad"])))
        return got
    if case["op"] == "orthogonalize":
        return [_exact_orthogonal(s["x"].double())]
    ws, vs = [], []
    for w, g, v, scale in zip(s["w"], s["g"], s["v"], s["scale"]):
        vs.append(MOMENTUM * v.double() - g.double())
        ws.append((1 - LR * DECAY) * w.double()
                  + LR * scale * _exact_orthogonal(vs[-1]))
    return [ws, vs, ws]
