"""Functional ops: CPU reference numerics + GPU autograd wrappers.

Conventions (both paths):
  * images are NHWC, channels padded to CPAD (16; stems 4) — see
    ``cpad_for``;
  * GPU compute dtype is bf16 with fp32 master weights / statistics;
    the CPU path runs fp32 and defines the semantics the HIP kernels in
    ``ops/hip/`` are tested against (tests/test_kernels_gpu.py).

The GPU conv/linear Functions live in models/layers.py next to their
layout state; this module holds the stateless ops (pool, LRN, BN,
dropout, relu, add, softmax-xent) and the CPU references for everything,
including conv (reference: the ops of Theano-MPI's layer library
``theanompi/models/layers2.py`` [pub]).
"""

import torch
import torch.nn.functional as F

from theanompi_amd import ops as _ops

# ---------------------------------------------------------------------------
# channel padding helpers
# ---------------------------------------------------------------------------

CPAD = 16


def cpad_for(c):
    """Physical channel count for a logical channel count."""
    if c <= 4:
        return 4
    return (c + CPAD - 1) // CPAD * CPAD


def pad_channels(x_nhwc, c_phys):
    """Zero-pad the last dim of an NHWC tensor to c_phys."""
    c = x_nhwc.shape[-1]
    if c == c_phys:
        return x_nhwc
    return F.pad(x_nhwc, (0, c_phys - c))


# ---------------------------------------------------------------------------
# CPU reference implementations (fp32, NHWC in/out)
# ---------------------------------------------------------------------------

def conv2d_ref(x, w_kcrs, bias, stride=(1, 1), pad=(0, 0), groups=1,
               relu=False):
    """x: [N,H,W,C] ; w: [K,C/G,R,S] ; returns [N,P,Q,K]."""
    xc = x.permute(0, 3, 1, 2).contiguous()
    y = F.conv2d(xc, w_kcrs, bias, stride=stride, padding=pad, groups=groups)
    y = y.permute(0, 2, 3, 1).contiguous()
    return F.relu(y) if relu else y


def linear_ref(x, w_in_out, bias, relu=False):
    """x: [B, IN]; w: [IN, OUT] (Theano layout)."""
    y = x @ w_in_out
    if bias is not None:
        y = y + bias
    return F.relu(y) if relu else y


def maxpool2d_ref(x, kernel, stride, pad=(0, 0)):
    xc = x.permute(0, 3, 1, 2)
    y = F.max_pool2d(xc, kernel, stride, pad)
    return y.permute(0, 2, 3, 1).contiguous()


def avgpool2d_ref(x, kernel, stride, pad=(0, 0)):
    xc = x.permute(0, 3, 1, 2)
    y = F.avg_pool2d(xc, kernel, stride, pad, count_include_pad=True)
    return y.permute(0, 2, 3, 1).contiguous()


def lrn_ref(x, size=5, alpha=1e-4, beta=0.75, k=1.0):
    """Cross-map LRN, AlexNet-style:  y = x * (k + alpha/size * sum x^2)^-beta
    over a window of `size` channels centred on c (clamped at the edges).
    Matches theano dnn LRN / F.local_response_norm semantics."""
    xc = x.permute(0, 3, 1, 2)
    y = F.local_response_norm(xc, size=size, alpha=alpha, beta=beta, k=k)
    return y.permute(0, 2, 3, 1).contiguous()


def batchnorm_ref(x, gamma, beta, running_mean, running_var, training,
                  momentum=0.1, eps=1e-5, relu=False):
    xc = x.permute(0, 3, 1, 2)
    y = F.batch_norm(xc, running_mean, running_var, gamma, beta,
                     training=training, momentum=momentum, eps=eps)
    y = y.permute(0, 2, 3, 1).contiguous()
    return F.relu(y) if relu else y


def dropout_ref(x, p, training):
    return F.dropout(x, p=p, training=training)


def softmax_xent_ref(logits, labels, n_classes=None):
    """logits [B, Cp] (maybe channel-padded), labels int64 [B].
    Returns (mean loss, probs [B, Cp]).  Padded columns are masked."""
    if n_classes is not None and n_classes < logits.shape[1]:
        mask = torch.full_like(logits, float("-inf"))
        mask[:, :n_classes] = 0.0
        logits = logits + mask
    probs = F.softmax(logits.float(), dim=1)
    loss = F.cross_entropy(logits.float(), labels)
    return loss, probs


def layernorm_ref(x, gamma, beta, eps=1e-5, n_features=None):
    """Normalisation over the last dimension's first ``n_features``
    channels, statistics in at least fp32; zeros behind them."""
    n = n_features or x.shape[-1]
    wide = torch.promote_types(x.dtype, torch.float32)
    xf = x[..., :n].to(wide)
    d = xf - xf.mean(dim=-1, keepdim=True)
    var = (d * d).mean(dim=-1, keepdim=True)
    y = d / torch.sqrt(var + eps) * gamma[:n] + beta[:n]
    return pad_channels(y, x.shape[-1]).to(x.dtype)


def label_logprobs_ref(logits, labels, n_classes=None, top=0):
    """See :func:`label_logprobs`."""
    n = n_classes or logits.shape[1]
    wide = torch.promote_types(logits.dtype, torch.float32)
    z = logits[:, :n].to(wide)
    masked = z == float("-inf")
    empty = masked.all(dim=1, keepdim=True)
    logp = torch.log_softmax(torch.where(empty, torch.zeros_like(z), z),
                             dim=1)
    p = logp.exp()
    entropy = -(p * logp.masked_fill(p == 0, 0.0)).sum(dim=1)
    entropy = entropy.masked_fill(empty[:, 0], 0.0)
    logp = logp.masked_fill(empty, float("-inf"))
    given = logp.gather(1, labels.clamp(0, n - 1)[:, None])[:, 0]
    given = given * torch.ones_like(given).masked_fill(labels >= n,
                                                       float("nan"))
    given = given.masked_fill(labels < 0, 0.0)
    # a stable sort leaves equal values in the order of their index
    best = z.detach().sort(dim=1, descending=True, stable=True)
    best = best.indices[:, :top].contiguous()
    return given, entropy, logp.gather(1, best), best


#: the quintic whose iteration takes singular values towards 1
NS_QUINTIC = (3.4445, -4.775, 2.0315)


def orthogonalize_ref(x, steps=5):
    """See :func:`orthogonalize`."""
    y = x.to(torch.promote_types(x.dtype, torch.float32))
    tall = y.shape[-2] > y.shape[-1]
    if tall:
        y = y.transpose(-2, -1)
    norm = y.double().square().sum(dim=(-2, -1), keepdim=True).sqrt()
    y = (y / (norm + 1e-7)).to(y.dtype)
    a, b, c = NS_QUINTIC
    for _ in range(steps):
        gram = y @ y.transpose(-2, -1)
        y = a * y + (b * gram + c * (gram @ gram)) @ y
    return (y.transpose(-2, -1) if tall else y).to(x.dtype).contiguous()


def muon_update_ref(w, g, v, out, keep, rate, momentum, phase, steps):
    """One matrix (or batch) of :func:`muon_update`."""
    if phase != 2:
        v.mul_(momentum).sub_(g)
    if phase != 1:
        w.mul_(keep).add_(orthogonalize_ref(v, steps), alpha=rate)
        if out is not None:
            out.copy_(w)


# ---------------------------------------------------------------------------
# GPU autograd wrappers (stateless ops). Each calls theanompi_amd._C.
# (layernorm and label_logprobs have their nodes there, in bindings.cpp.)
# ---------------------------------------------------------------------------

class _MaxPool2dFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, kernel, stride, pad):
        C = _ops.ext()
        kh, kw = kernel
        sh, sw = stride
        ph, pw = pad
        xp = C.halo_pad(x, ph, pw, float("-inf")) if (ph or pw) else x
        n, hp, wp, c = xp.shape
        p = (hp - kh) // sh + 1
        q = (wp - kw) // sw + 1
        y = torch.empty((n, p, q, c), dtype=x.dtype, device=x.device)
        argmax = torch.empty((n, p, q, c), dtype=torch.uint8, device=x.device)
        C.maxpool_fwd(xp, y, argmax, kh, kw, sh, sw)
        ctx.save_for_backward(argmax)
        ctx.meta = (x.shape, kernel, stride, pad)
        return y

    @staticmethod
    def backward(ctx, dy):
        (argmax,) = ctx.saved_tensors
        xshape, kernel, stride, pad = ctx.meta
        C = _ops.ext()
        # maxpool_bwd_k writes every dx element - no pre-zero needed
        dx = torch.empty(xshape, dtype=dy.dtype, device=dy.device)
        C.maxpool_bwd(dy.contiguous(), argmax, dx,
                      kernel[0], kernel[1], stride[0], stride[1],
                      pad[0], pad[1])
        return dx, None, None, None


class _AvgPool2dFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, kernel, stride, pad):
        C = _ops.ext()
        kh, kw = kernel
        sh, sw = stride
        ph, pw = pad
        xp = C.halo_pad(x, ph, pw, 0.0) if (ph or pw) else x
        n, hp, wp, c = xp.shape
        p = (hp - kh) // sh + 1
        q = (wp - kw) // sw + 1
        y = torch.empty((n, p, q, c), dtype=x.dtype, device=x.device)
        C.avgpool_fwd(xp, y, kh, kw, sh, sw)
        ctx.meta = (x.shape, kernel, stride, pad)
        return y

    @staticmethod
    def backward(ctx, dy):
        xshape, kernel, stride, pad = ctx.meta
        C = _ops.ext()
        dx = torch.empty(xshape, dtype=dy.dtype, device=dy.device)
        C.avgpool_bwd(dy.contiguous(), dx, kernel[0], kernel[1],
                      stride[0], stride[1], pad[0], pad[1])
        return dx, None, None, None


class _LRNFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, size, alpha, beta, k):
        C = _ops.ext()
        y = torch.empty_like(x)
        # 1/denom in bf16: halves the save traffic, and backward
        # reconstructs x from y so only (y, scale) need saving at all
        scale = torch.empty(x.shape, dtype=torch.bfloat16,
                            device=x.device)
        C.lrn_fwd(x, y, scale, size, alpha, beta, k)   # scale = 1/denom
        ctx.save_for_backward(y, scale)
        ctx.meta = (size, alpha, beta, k)
        return y

    @staticmethod
    def backward(ctx, dy):
        y, scale = ctx.saved_tensors
        size, alpha, beta, k = ctx.meta
        C = _ops.ext()
        dx = torch.empty_like(y)
        C.lrn_bwd(dy.contiguous(), y, scale, dx, size, alpha, beta, k)
        return dx, None, None, None, None


class _BatchNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gamma, beta, running_mean, running_var,
                training, momentum, eps, relu, prestats=None,
                residual=None):
        # residual: fused residual join y = [relu](bn(x) + residual) —
        # one pass instead of bn_apply + add_relu (ResNet bottleneck
        # exits; the separate adds were ~8% of its step)
        C = _ops.ext()
        y = torch.empty_like(x)
        c = x.shape[-1]
        save_mean = torch.empty(c, dtype=torch.float32, device=x.device)
        save_invstd = torch.empty(c, dtype=torch.float32, device=x.device)
        C.bn_fwd(x, gamma, beta, y, save_mean, save_invstd,
                 running_mean, running_var, float(momentum), float(eps),
                 bool(training), bool(relu), prestats,
                 residual.contiguous() if residual is not None else None)
        ctx.save_for_backward(x, gamma, beta, save_mean, save_invstd, y)
        ctx.relu = relu
        ctx.training = training
        ctx.has_res = residual is not None
        return y

    @staticmethod
    def backward(ctx, dy):
        x, gamma, beta, save_mean, save_invstd, y = ctx.saved_tensors
        C = _ops.ext()
        dx = torch.empty_like(x)
        dgamma = torch.empty_like(gamma)
        dbeta = torch.empty_like(gamma)
        dy = dy.contiguous()
        dres = None
        if ctx.has_res and ctx.relu:
            # masked dy comes out of the same kernel pass
            dres = torch.empty_like(dy)
        C.bn_bwd(dy, x, gamma, beta, save_mean,
                 save_invstd, y, dx, dgamma, dbeta, bool(ctx.relu),
                 dres, bool(ctx.has_res))
        if ctx.has_res and not ctx.relu:
            dres = dy              # pass-through, no kernel needed
        return (dx, dgamma, dbeta, None, None, None, None, None, None,
                None, dres)


class _ReluFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        C = _ops.ext()
        y = torch.empty_like(x)
        C.relu_fwd(x, y)
        ctx.save_for_backward(y)
        return y

    @staticmethod
    def backward(ctx, dy):
        (y,) = ctx.saved_tensors
        C = _ops.ext()
        dx = torch.empty_like(dy)
        C.relu_bwd(dy.contiguous(), y, dx)
        return dx


class _AddFn(torch.autograd.Function):
    """Residual add (+ optional relu) for ResNet."""
    @staticmethod
    def forward(ctx, a, b, relu):
        C = _ops.ext()
        y = torch.empty_like(a)
        C.add_relu(a, b, y, bool(relu))
        ctx.relu = relu
        if relu:
            ctx.save_for_backward(y)
        return y

    @staticmethod
    def backward(ctx, dy):
        if ctx.relu:
            (y,) = ctx.saved_tensors
            C = _ops.ext()
            dx = torch.empty_like(dy)
            C.relu_bwd(dy.contiguous(), y, dx)
            return dx, dx, None
        return dy, dy, None


class _DropoutFn(torch.autograd.Function):
    _seed_buf = {}

    @staticmethod
    def _seed(device):
        t = _DropoutFn._seed_buf.get(device)
        if t is None:
            t = torch.tensor([12345], dtype=torch.int64, device=device)
            _DropoutFn._seed_buf[device] = t
        return t

    @staticmethod
    def forward(ctx, x, p):
        C = _ops.ext()
        y = torch.empty_like(x)
        mask = torch.empty(x.shape, dtype=torch.uint8, device=x.device)
        # device-resident seed (bumped in-kernel) keeps masks fresh under
        # hipGraph replay
        C.dropout_fwd(x, y, mask, float(p), _DropoutFn._seed(x.device))
        ctx.save_for_backward(mask)
        ctx.p = p
        return y

    @staticmethod
    def backward(ctx, dy):
        (mask,) = ctx.saved_tensors
        C = _ops.ext()
        dx = torch.empty_like(dy)
        C.dropout_bwd(dy.contiguous(), mask, dx, float(ctx.p))
        return dx, None


class _SoftmaxXentFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, n_classes):
        C = _ops.ext()
        b = logits.shape[0]
        probs = torch.empty_like(logits)
        loss = torch.empty(b, dtype=torch.float32, device=logits.device)
        # fused batch reductions: stats = [sum(loss), count(top1 err)],
        # accumulated by the kernel's per-row atomics — no torch
        # mean/argmax glue in the train step
        stats = torch.zeros(2, dtype=torch.float32, device=logits.device)
        C.softmax_xent_fwd(logits, labels, probs, loss, int(n_classes),
                           stats)
        ctx.save_for_backward(probs, labels)
        ctx.n_classes = n_classes
        sm = stats * (1.0 / b)
        # probs/err are inference-only outputs: backward below only
        # accounts for dloss, so autograd must not route gradients
        # through them silently
        ctx.mark_non_differentiable(probs)
        err = sm[1]
        ctx.mark_non_differentiable(err)
        return sm[0], probs, err

    @staticmethod
    def backward(ctx, dloss, dprobs, derr):
        probs, labels = ctx.saved_tensors
        C = _ops.ext()
        dlogits = torch.empty_like(probs)
        scale = 1.0 / probs.shape[0]
        C.softmax_xent_bwd(probs, labels, dlogits, scale, int(ctx.n_classes))
        if dloss.numel() == 1:
            dlogits = dlogits * dloss.to(dlogits.dtype)  # no host sync
        return dlogits, None, None


# ---------------------------------------------------------------------------
# public dispatchers
# ---------------------------------------------------------------------------

def _pair(v):
    return (v, v) if isinstance(v, int) else tuple(v)


def maxpool2d(x, kernel, stride, pad=0):
    kernel, stride, pad = _pair(kernel), _pair(stride), _pair(pad)
    if x.is_cuda:
        return _MaxPool2dFn.apply(x, kernel, stride, pad)
    return maxpool2d_ref(x, kernel, stride, pad)


def avgpool2d(x, kernel, stride, pad=0):
    kernel, stride, pad = _pair(kernel), _pair(stride), _pair(pad)
    if x.is_cuda:
        return _AvgPool2dFn.apply(x, kernel, stride, pad)
    return avgpool2d_ref(x, kernel, stride, pad)


def lrn(x, size=5, alpha=1e-4, beta=0.75, k=1.0):
    if x.is_cuda:
        return _LRNFn.apply(x, size, alpha, beta, k)
    return lrn_ref(x, size, alpha, beta, k)


def batchnorm(x, gamma, beta, running_mean, running_var, training,
              momentum=0.1, eps=1e-5, relu=False, prestats=None,
              residual=None):
    if x.is_cuda:
        return _BatchNormFn.apply(x, gamma, beta, running_mean,
                                  running_var, training, momentum, eps,
                                  relu, prestats, residual)
    y = batchnorm_ref(x, gamma.float(), beta.float(), running_mean,
                      running_var, training, momentum, eps, relu=False)
    if residual is not None:
        y = y + residual
    return F.relu(y) if relu else y


def relu(x):
    if x.is_cuda:
        return _ReluFn.apply(x)
    return F.relu(x)


def add(a, b, relu=False):
    if a.is_cuda:
        return _AddFn.apply(a, b, relu)
    y = a + b
    return F.relu(y) if relu else y


def dropout(x, p, training):
    if not training or p == 0.0:
        return x
    if x.is_cuda:
        return _DropoutFn.apply(x, p)
    return F.dropout(x, p=p, training=True)


def softmax_xent(logits, labels, n_classes=None):
    """Fused softmax + cross-entropy.  Returns (mean_loss, probs)."""
    n_classes = n_classes or logits.shape[1]
    if logits.is_cuda:
        loss, probs, _err = _SoftmaxXentFn.apply(logits, labels, n_classes)
        return loss, probs
    return softmax_xent_ref(logits, labels, n_classes)


def softmax_xent_err(logits, labels, n_classes=None):
    """softmax_xent plus the fused top-1 training error: on GPU the
    loss mean AND the err count ride the xent kernel's atomics, so the
    train step needs no torch argmax/mean glue.  Returns
    (mean_loss, probs, err)."""
    n_classes = n_classes or logits.shape[1]
    if logits.is_cuda:
        return _SoftmaxXentFn.apply(logits, labels, n_classes)
    loss, probs = softmax_xent_ref(logits, labels, n_classes)
    with torch.no_grad():
        pred = logits[:, :n_classes].argmax(dim=1)
        err = (pred != labels).float().mean()
    return loss, probs, err


def _check_float(t, name):
    ok = (torch.float32, torch.float16, torch.bfloat16)
    if t.dtype not in ok and (t.is_cuda or t.dtype != torch.float64):
        raise TypeError(f"{name} must be float32, float16 or bfloat16, "
                        f"not {t.dtype}")


def _check_count(n, most, name):
    if n is None:
        return most
    if isinstance(n, bool) or not isinstance(n, int) or not 1 <= n <= most:
        raise ValueError(f"{name} must be a whole number from 1 to {most}, "
                         f"not {n!r}")
    return n


def layernorm(x, gamma, beta, eps=1e-5, n_features=None):
    """Layer normalisation over the last (channel) dimension.

    ``x``: [..., C] in float32, float16 or bfloat16; rows may lie apart
    (a channel slice of a wider buffer).  ``gamma``, ``beta``: float32
    [C].  Only the first ``n_features`` channels count (default: all);
    the physical padding behind them is not read, its outputs and
    gradients are 0.  Statistics are kept in float32.  Returns x's shape
    and type.  On the GPU a row may have 2^28 channels.  Differentiable once
    in x, gamma and beta; the sums of the latter two have a fixed order, so a
    repeated call gives the same bits."""
    _check_float(x, "x")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("x needs at least one channel")
    c = x.shape[-1]
    for t, name in ((gamma, "gamma"), (beta, "beta")):
        if t.shape != (c,):
            raise ValueError(f"{name} must have shape ({c},), "
                             f"not {tuple(t.shape)}")
        if t.dtype != (torch.float64 if x.dtype == torch.float64
                       else torch.float32):
            raise TypeError(f"{name} must be float32, not {t.dtype}")
        if t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, x on {x.device}")
    eps = float(eps)
    if not 0.0 <= eps < float("inf"):
        raise ValueError(f"eps must not be negative, not {eps}")
    n = _check_count(n_features, c, "n_features")
    if x.is_cuda:
        return _ops.ext().layernorm(x, gamma.contiguous(),
                                    beta.contiguous(), eps, n)
    return layernorm_ref(x, gamma, beta, eps, n)


#: alternatives that label_logprobs can name
TOP_MAX = 32


def label_logprobs(logits, labels, n_classes=None, top=0):
    """Log probability of each row's given class, the entropy of the
    row's distribution, and its most probable classes.

    ``logits``: [B, C] in float32, float16 or bfloat16, of which the
    first ``n_classes`` columns count; rows may lie apart.  ``labels``:
    int64 [B]; below 0: no class is given (log probability 0), from
    ``n_classes`` on: NaN.  Returns (logp [B], entropy [B], top_logp
    [B, top], top_idx [B, top]): float32, and int64 class numbers, best
    first, equal logits by ascending class.  Logits of -inf are masked
    classes: probability 0, and no gradient unless the label or an
    alternative names them.  A row of masked classes alone has logp
    -inf, entropy 0 and gradient 0.  A NaN or +inf gives
    NaN in its row.  On the GPU a row may have 2^21 classes in float32,
    2^22 in the 16-bit types.  Differentiable once in the logits, through
    logp, entropy and top_logp."""
    _check_float(logits, "logits")
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError("logits must be [rows, classes], not "
                         f"{tuple(logits.shape)}")
    if labels.dtype != torch.int64:
        raise TypeError(f"labels must be int64, not {labels.dtype}")
    if labels.shape != logits.shape[:1]:
        raise ValueError(f"labels must have shape ({logits.shape[0]},), "
                         f"not {tuple(labels.shape)}")
    if labels.device != logits.device:
        raise ValueError(f"labels are on {labels.device}, logits on "
                         f"{logits.device}")
    n = _check_count(n_classes, logits.shape[1], "n_classes")
    if isinstance(top, bool) or not isinstance(top, int) \
            or not 0 <= top <= min(n, TOP_MAX):
        raise ValueError(f"top must be a whole number from 0 to "
                         f"{min(n, TOP_MAX)}, not {top!r}")
    if logits.is_cuda:
        return tuple(_ops.ext().label_logprobs(
            logits, labels.contiguous(), n, top))
    return label_logprobs_ref(logits, labels, n, top)


def _check_steps(steps):
    if isinstance(steps, bool) or not isinstance(steps, int) \
            or not 1 <= steps <= 64:
        raise ValueError("steps must be a whole number from 1 to 64, "
                         f"not {steps!r}")


def orthogonalize(x, steps=5):
    """Newton-Schulz products that take the singular values of a matrix
    towards 1 (into about 0.7 to 1.2) and leave its singular vectors.

    ``x``: [rows, cols] or [batch, rows, cols] in float32, float16 or
    bfloat16.  X = x / (|x|_F + 1e-7), then ``steps`` times
    X <- (a + b XX^T + c (XX^T)^2) X with (a, b, c) = NS_QUINTIC, on the
    orientation that has the smaller XX^T.  On the GPU products keep 22 bits
    of their operands and add up in float32, for all types: five steps are
    off by some 1e-6 of the result's norm, less than plain float32 products
    are from 65 rows on, and up to about twice that of fewer.  Returns a new
    tensor of x's shape and type, without a gradient."""
    _check_float(x, "x")
    if x.dim() not in (2, 3):
        raise ValueError("x must be [rows, cols] or [batch, rows, cols], "
                         f"not {tuple(x.shape)}")
    _check_steps(steps)
    with torch.no_grad():
        x = x.detach()
        if x.is_cuda:
            return _ops.ext().orthogonalize(x, steps)
        return orthogonalize_ref(x, steps) if x.numel() else x.clone()


def _check_apart(written, read):
    """No memory of ``written`` is another's, or any of ``read``'s (on the
    GPU the extension looks)."""
    end = write_end = 0
    for start, stop, writes in sorted(
            (t.data_ptr(), t.data_ptr() + t.nbytes, writes)
            for ts, writes in ((written, True), (read, False))
            for t in ts if t.numel()):
        if start < (end if writes else write_end):
            raise ValueError("a weight, momentum or working copy shares "
                             "memory with another tensor of the list")
        end = max(end, stop)
        if writes:
            write_end = max(write_end, stop)


def muon_update(ws, gs, vs, outs, lrs, wds, momentum, scales, phase=0,
                steps=5):
    """Orthogonalised momentum update of a list of weights, in place:

      v = momentum*v - g;   w = (1 - lr*wd)*w + lr*scale*orthogonalize(v)

    ``ws``, ``gs``, ``vs``: float32, contiguous, [rows, cols] or [batch,
    rows, cols] (each matrix of a batch on its own); ``outs``: bf16
    working copies of w, or None in the place of one that is not kept.
    Weights, momenta and copies share no memory with anything in the list.
    ``phase``: 0 the whole update, 1 the momentum only, 2 the weights
    only (gs are not read and may be None), as in the SGD step.  On the GPU
    every matrix of the list goes through each product in one launch, and
    what its sums are cut into depends on the list: equal calls give equal
    bits, other lists round a matrix otherwise."""
    many = len(ws)
    for name, part in (("gs", gs), ("vs", vs), ("outs", outs),
                       ("lrs", lrs), ("wds", wds), ("scales", scales)):
        if len(part) != many:
            raise ValueError(f"{name} has {len(part)} entries, ws {many}")
    if phase not in (0, 1, 2):
        raise ValueError(f"phase must be 0, 1 or 2, not {phase!r}")
    _check_steps(steps)
    if not many:
        return
    for i in range(many):
        w = ws[i]
        parts = [("w", w), ("v", vs[i])]
        if phase != 2:
            parts.append(("g", gs[i]))
        for name, t in parts:
            if t.dtype != torch.float32:
                raise TypeError(f"{name} {i} must be float32, "
                                f"not {t.dtype}")
            if not t.is_contiguous() or t.shape != w.shape \
                    or t.dim() not in (2, 3):
                raise ValueError(
                    f"{name} {i} must be a contiguous [rows, cols] or "
                    "[batch, rows, cols] of its weight's shape")
            if t.device != ws[0].device:
                raise ValueError(f"{name} {i} is on {t.device}, the first "
                                 f"weight on {ws[0].device}")
        if outs[i] is not None:
            if outs[i].dtype != torch.bfloat16:
                raise TypeError(f"out {i} must be bfloat16, "
                                f"not {outs[i].dtype}")
            if not outs[i].is_contiguous() \
                    or outs[i].numel() != w.numel() \
                    or outs[i].device != w.device:
                raise ValueError(f"out {i} must be contiguous, of its "
                                 "weight's size and on its device")
    keeps = [1.0 - lr * wd for lr, wd in zip(lrs, wds)]
    rates = [lr * scale for lr, scale in zip(lrs, scales)]
    with torch.no_grad():
        if ws[0].is_cuda:
            none = torch.empty(0, dtype=torch.bfloat16,
                               device=ws[0].device)
            _ops.ext().muon_update(
                [w.detach() for w in ws],
                [none if phase == 2 else g for g in gs], list(vs),
                [none if o is None else o for o in outs], keeps, rates,
                float(momentum), phase, steps)
            return
        _check_apart([*ws, *vs, *(o for o in outs if o is not None)],
                     gs if phase != 2 else [])
        for i in range(many):
            out = outs[i]
            if ws[i].numel():
                muon_update_ref(ws[i], gs[i], vs[i],
                                out if out is None else out.view_as(ws[i]),
                                keeps[i], rates[i], momentum, phase, steps)
