"""Layer norm, class log probabilities, the orthogonalised update: the
CPU forms against elementary formulas in 64 bits, the HIP kernels against
the CPU forms in 64 bits, on the same inputs.

Tolerances count roundings: half a step of the output's type on the
result, and DEPTH steps of fp32 (2^-24 each) on the magnitudes that are
added up.  DEPTH = 128 covers the longest chain of additions any of the
reductions here has: at most 64 values in a lane, 6 exchanges in a wave,
16 waves, and as many again for a second stage."""

import math

import pytest
import torch

from theanompi_amd.ops import functional as OF

gpu = pytest.mark.gpu
U = 2.0 ** -24
DEPTH = 128
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def half(t):
    return torch.finfo(t).eps / 2


def dev():
    return torch.device("cuda", 0)


def close(got, ref, tol, what=""):
    """|got - ref| <= tol everywhere (64 bits), NaN and infinities alike."""
    got, ref = got.detach().double().cpu(), ref.detach().double().cpu()
    tol = torch.as_tensor(tol, dtype=torch.float64).cpu().expand(ref.shape)
    assert got.shape == ref.shape, what
    fine = torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), what
    inf = torch.isinf(ref)
    assert torch.equal(got[inf], ref[inf]), what
    off = (got - ref).abs()[fine]
    bad = off > tol[fine]
    assert not bad.any(), (
        f"{what}: {int(bad.sum())} of {ref.numel()} off, worst "
        f"{float((off / tol[fine].clamp_min(1e-300)).max()):.2f} times "
        "the tolerance")


# ---------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------

def ln_formula(x, gamma, beta, dy, eps, n):
    """Outputs in 64 bits and, for each, what roundings scale with."""
    c = x.shape[-1]
    x, dy = x.double().reshape(-1, c)[:, :n], dy.double().reshape(-1, c)
    dy = dy[:, :n]
    gamma, beta = gamma.double()[:n], beta.double()[:n]
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
    xh = (x - mean) * rstd
    g = dy * gamma
    c1, c2 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    out = [xh * gamma + beta, rstd * (g - c1 - xh * c2),
           (dy * xh).sum(0), dy.sum(0)]
    # an error of xh: of the mean and of the difference, and relative
    exh = DEPTH * U * (rstd * (x.abs().amax(1, keepdim=True)) + xh.abs())
    a1, a2 = g.abs().mean(1, keepdim=True), (g * xh).abs().mean(
        1, keepdim=True)
    a3 = (g.abs() * exh).mean(1, keepdim=True)
    tol = [gamma.abs() * exh + 4 * U * (out[0].abs() + beta.abs()),
           rstd * (exh * c2.abs() + xh.abs() * (a3 + DEPTH * U * a2)
                   + DEPTH * U * (g.abs() + a1))
           + DEPTH * U * out[1].abs(),
           (dy.abs() * exh).sum(0) + DEPTH * U * (dy * xh).abs().sum(0),
           DEPTH * U * dy.abs().sum(0)]
    return out, tol


def ln_check(x, gamma, beta, dy, n=None, eps=1e-5):
    c = x.shape[-1]
    leaves = [t.detach().requires_grad_(True) for t in (x, gamma, beta)]
    y = OF.layernorm(*leaves, eps=eps, n_features=n)
    assert y.shape == x.shape and y.dtype == x.dtype
    got = [y, *torch.autograd.grad(y, leaves, dy)]
    n = n or c
    ref, tol = ln_formula(x, gamma, beta, dy, eps, n)
    for i, name in enumerate(("y", "dx", "dgamma", "dbeta")):
        a = got[i].reshape(-1, c) if i < 2 else got[i]
        assert torch.equal(a[..., n:].float(),
                           torch.zeros_like(a[..., n:]).float()), name
        t = tol[i] + (half(x.dtype) * ref[i].abs() if i < 2 else 0)
        # below its normal numbers a type's step no longer shrinks
        close(a[..., :n], ref[i], t + torch.finfo(a.dtype).tiny, name)
    return got


def ln_inputs(shape, dtype, device, seed=0, offset=0.5):
    g = torch.Generator().manual_seed(seed)
    c = shape[-1]
    x = (torch.randn(*shape, generator=g) * 1.5 + offset).to(dtype)
    gamma = 1 + 0.3 * torch.randn(c, generator=g)
    beta = 0.2 * torch.randn(c, generator=g)
    dy = torch.randn(*shape, generator=g).to(dtype)
    return [t.to(device) for t in (x, gamma, beta, dy)]


@pytest.mark.parametrize("shape,n", [((5, 7), None), ((3, 2, 16), 10),
                                     ((1, 1), None), ((0, 4), None)])
def test_layernorm_cpu(shape, n):
    for dtype in TYPES:
        ln_check(*ln_inputs(shape, dtype, "cpu"), n=n)


def test_layernorm_gradient_against_differences():
    x, gamma, beta, _ = [t.double().requires_grad_(True) for t in
                         ln_inputs((3, 6), torch.float32, "cpu")]
    assert torch.autograd.gradcheck(
        lambda *a: OF.layernorm(*a, n_features=5), (x, gamma, beta))


LN_SHAPES = [(1, 1), (1, 3), (7, 8), (33, 64), (5, 65), (2, 3, 127),
             (260, 128), (31, 256), (70, 257), (600, 300), (513, 512),
             (129, 1000), (40, 1001), (19, 2048), (11, 2049), (6, 4096),
             (5, 8191), (4, 16384), (3, 16385), (2, 33000), (2, 2, 5, 48),
             (5000, 16), (700, 9001), (530, 20000), (520, 768), (6, 1500),
             (5, 2500), (600, 5000), (3, 12000)]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", LN_SHAPES, ids=str)
def test_layernorm_gpu(shape, dtype):
    ln_check(*ln_inputs(shape, dtype, dev()))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,n", [((9, 16), 1), ((9, 16), 10),
                                     ((700, 1008), 1000), ((3, 20000), 19),
                                     ((2, 40000), 39990)], ids=str)
def test_layernorm_gpu_padded_channels(shape, n, dtype):
    x, gamma, beta, dy = ln_inputs(shape, dtype, dev())
    for t in (x, gamma, beta, dy):      # never read
        t[..., n:] = float("nan")
    ln_check(x, gamma, beta, dy, n=n)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_layernorm_gpu_strides(dtype):
    x, gamma, beta, dy = ln_inputs((4, 6, 80), dtype, dev())
    # a channel slice at an odd element: rows 16-byte vectors do not meet
    xs, dys = x[..., 3:38], dy[..., 1:36]
    ln_check(xs, gamma[3:38], beta[3:38], dys)
    # channels apart, batch dimensions in another order, one row repeated
    for t, d in ((x.transpose(1, 2), dy.transpose(1, 2)),
                 (x.transpose(0, 1), dy.transpose(0, 1)),
                 (x[:1].expand(4, -1, -1), dy[:, :1].expand(-1, 6, -1))):
        c = t.shape[-1]
        g = torch.ones(c, device=dev()) * 1.25
        ln_check(t, g, g - 1, d)


@gpu
def test_layernorm_gpu_large_mean():
    # a spread far below the mean: squares of the values would lose it
    ln_check(*ln_inputs((64, 512), torch.float32, dev(), offset=1000.0))


@gpu
def test_layernorm_gpu_constant_rows_and_no_rows():
    x = torch.full((5, 64), 3.0, device=dev())
    gamma, beta = torch.ones(64, device=dev()), torch.ones(64, device=dev())
    assert torch.equal(OF.layernorm(x, gamma, beta), torch.ones_like(x))
    empty = torch.empty(0, 64, device=dev(), requires_grad=True)
    gamma.requires_grad_(True)
    y = OF.layernorm(empty, gamma, beta)
    dx, dgamma = torch.autograd.grad(y.sum(), (empty, gamma))
    assert dx.shape == (0, 64) and not dgamma.any()


@gpu
@pytest.mark.parametrize("dtype,value", [
    (torch.float32, 1000.0), (torch.float32, 16000.0), (torch.float32, 1e5),
    (torch.float32, -0.1), (torch.float16, 16000.0), (torch.float16, 1001.0),
    (torch.bfloat16, 1.5e5)])
def test_layernorm_gpu_rows_of_one_large_value(dtype, value):
    """Outputs are beta, at any width.  The mean as first summed is off by
    DEPTH U |x| at most; the mean of the deviations from it gives that to
    within DEPTH U again, (DEPTH U)^2 |x| = 6e-11 |x|, which is below half
    a step of x, so the mean is x.  The variance is off by 2 DEPTH U
    (DEPTH U x)^2 at most, dx by half of that relative to eps, and rounded."""
    for c in (3, 7, 48, 100, 300, 700, 1000, 1500, 2500, 5000, 9001, 12000,
              20000, 40000):
        for rows in (5, 600):
            _, gamma, beta, dy = ln_inputs((rows, c), dtype, dev())
            x = torch.full((rows, c), value, dtype=dtype, device=dev())
            leaf = x.requires_grad_(True)
            y = OF.layernorm(leaf, gamma, beta)
            assert torch.equal(y, beta.to(dtype).expand_as(y)), (c, rows)
            if abs(value) > 1001:
                continue
            (dx,) = torch.autograd.grad(y, leaf, dy)
            g = dy.double() * gamma.double()
            want = (g - g.mean(1, keepdim=True)) / math.sqrt(1e-5)
            var = 2 * DEPTH * U * (DEPTH * U * value) ** 2 / 1e-5
            close(dx, want, (var / 2 + DEPTH * U + half(dtype)) * want.abs()
                  + DEPTH * U * g.abs().mean(1, keepdim=True)
                  / math.sqrt(1e-5), (c, rows))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layernorm_gpu_overflowing_squares(dtype):
    """Deviations whose squares fp32 does not hold: the variance is infinite
    and outputs are beta, as in the CPU's form."""
    for c in (20, 1000, 20000):
        x, gamma, beta, _ = ln_inputs((4, c), torch.float32, dev())
        for t in (x * 1e25 + 1e30, x * 1e24, torch.full_like(x, 1.1e33)):
            t = t.to(dtype)
            y = OF.layernorm(t, gamma, beta)
            assert torch.equal(y, beta.to(dtype).expand_as(y)), c
            assert torch.equal(OF.layernorm(t.cpu(), gamma.cpu(),
                                            beta.cpu()), y.cpu())


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 2, 4, 16, 64, 256, 1024, 4096, 16384])
def test_layernorm_gpu_gradient_of_large_constant_rows(n, dtype):
    """Powers of two sum exactly: deviations are 0, 1/std is 1e15, and
    nothing behind the row's end may count (0 - 2^90 times 1e15 overflows
    there).  dx is (g - mean g) 1e15, off by the roundings of a sum."""
    for more in (0, 1, 3, 21, 300):
        for rows in (5, 600):
            c = n + more
            x = torch.full((rows, c), 2.0 ** 90, dtype=dtype, device=dev())
            _, gamma, beta, dy = ln_inputs((rows, c), dtype, dev())
            leaf = x.requires_grad_(True)
            ga = gamma.requires_grad_(True)
            y = OF.layernorm(leaf, ga, beta, eps=1e-30, n_features=n)
            dx, dgamma = torch.autograd.grad(y, (leaf, ga), dy)
            g = dy.double()[:, :n] * gamma.detach().double()[:n]
            want = (g - g.mean(1, keepdim=True)) * 1e15
            tol = (DEPTH * U + half(dtype)) * want.abs() + DEPTH * U * (
                g.abs() + g.abs().mean(1, keepdim=True)) * 1e15
            close(dx[:, :n], want, tol, (c, rows))
            assert not dx[:, n:].float().any() and not dgamma.any()


@gpu
@pytest.mark.parametrize("shape", [(700, 300), (100, 4000)], ids=str)
def test_layernorm_gpu_same_bits_again(shape):
    args = ln_inputs(shape, torch.bfloat16, dev())
    first, again = ln_check(*args), ln_check(*args)
    for a, b in zip(first, again):
        assert torch.equal(a, b)


@gpu
def test_layernorm_gpu_nan_stays_in_its_row():
    x, gamma, beta, _ = ln_inputs((8, 100), torch.bfloat16, dev())
    x[3, 7] = float("nan")
    x[5, 2] = float("inf")
    y = OF.layernorm(x, gamma, beta)
    assert torch.isnan(y[3]).all() and torch.isnan(y[5]).all()
    assert torch.isfinite(y[[0, 1, 2, 4, 6, 7]]).all()


@gpu
@pytest.mark.parametrize("rows", [5, 700])
def test_layernorm_gpu_nan_leaves_padded_channels_alone(rows):
    x, gamma, beta, dy = ln_inputs((rows, 48), torch.bfloat16, dev())
    x[0, 3] = float("nan")
    leaves = [t.requires_grad_(True) for t in (x, gamma, beta)]
    y = OF.layernorm(*leaves, n_features=40)
    for g in (y, *torch.autograd.grad(y, leaves, dy)):
        assert not g[..., 40:].float().any()


def test_layernorm_refusals():
    x, gamma, beta, _ = ln_inputs((4, 8), torch.float32, "cpu")
    for bad in (torch.ones(4, 8, dtype=torch.int32), x.to(torch.complex64)):
        with pytest.raises(TypeError):
            OF.layernorm(bad, gamma, beta)
    with pytest.raises(TypeError):
        OF.layernorm(x, gamma.half(), beta)
    for g in (gamma[:7], gamma[None]):
        with pytest.raises(ValueError):
            OF.layernorm(x, g, beta)
        with pytest.raises(ValueError):
            OF.layernorm(x, gamma, g)
    for n in (0, -1, 9, 2.0, True):
        with pytest.raises(ValueError):
            OF.layernorm(x, gamma, beta, n_features=n)
    for eps in (-1e-5, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            OF.layernorm(x, gamma, beta, eps=eps)
    with pytest.raises(ValueError):
        OF.layernorm(torch.empty(3, 0), torch.empty(0), torch.empty(0))
    with pytest.raises(ValueError):
        OF.layernorm(torch.tensor(1.0), gamma, beta)
    with pytest.raises(ValueError):
        OF.layernorm(x, gamma.to("meta"), beta)


# ---------------------------------------------------------------------------
# class log probabilities
# ---------------------------------------------------------------------------

def lp_formula(x, labels, n, k, grads):
    """Outputs and dlogits in 64 bits, row by row from the definition,
    and what roundings scale with."""
    x = x.double()[:, :n]
    rows = x.shape[0]
    logp, ent = torch.zeros(rows), torch.zeros(rows)
    logp, ent = logp.double(), ent.double()
    top, idx = torch.zeros(rows, k).double(), torch.zeros(rows, k).long()
    dx, tl, te = torch.zeros_like(x), logp.clone(), ent.clone()
    tt, td = top.clone(), dx.clone()
    dl, dh, dt = [g.double() for g in grads]
    for r in range(rows):
        v, lab = x[r], int(labels[r])
        best = torch.sort(v, descending=True, stable=True).indices[:k]
        idx[r] = best
        if (v == -math.inf).all():
            logp[r] = 0.0 if lab < 0 else -math.inf
            top[r] = -math.inf
            continue
        lp = v - torch.logsumexp(v, 0)
        p = lp.exp()
        zlp = torch.where(p > 0, lp, torch.zeros_like(lp))
        h = -(p * zlp).sum()
        ent[r], top[r] = h, lp[best]
        logp[r] = 0.0 if lab < 0 else lp[lab]
        total = dt[r].sum() + (dl[r] if lab >= 0 else 0.0)
        coef = -total - dh[r] * (zlp + h)
        dx[r] = p * coef
        if lab >= 0:
            dx[r, lab] += dl[r]
        dx[r, best] += dt[r]
        # logits enter as differences from the maximum; an exponential
        # is off by its argument's rounding
        spread = (p * zlp.abs()).sum() + 1
        e = DEPTH * U * spread
        fin = torch.where(torch.isfinite(v), v, torch.zeros_like(v)).abs()
        tl[r] = e + 4 * U * (fin[max(lab, 0)] + fin.max())
        te[r] = 2 * e * spread
        tt[r] = e + 4 * U * (fin[best] + fin.max())
        w = dt[r].abs().sum() + dl[r].abs() + dh[r].abs() * (
            zlp.abs() + h.abs() + 1)
        # fp32 probabilities below its smallest normal number, 2^-126,
        # may be taken as 0: p is off by up to that, its product with the
        # coefficient by that times w
        td[r] = (p * w * (2 * e + DEPTH * U * (1 + zlp.abs()))
                 + 2.0 ** -126 * w)
        td[r] += 4 * U * dx[r].abs()
        if lab >= 0:
            td[r, lab] += 4 * U * dl[r].abs()
        td[r, best] += 4 * U * (dt[r].abs() + dl[r].abs())
    return (logp, ent, top, idx, dx), (tl, te, tt, None, td)


def lp_grads(rows, k, seed=1):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(rows, generator=g), torch.randn(rows, generator=g),
            torch.randn(rows, k, generator=g)]


def lp_check(x, labels, n=None, k=0):
    rows, c = x.shape
    grads = lp_grads(rows, k)
    leaf = x.detach().requires_grad_(True)
    out = OF.label_logprobs(leaf, labels, n_classes=n, top=k)
    assert [t.dtype for t in out] == [torch.float32] * 3 + [torch.int64]
    (dx,) = torch.autograd.grad(out[:3], leaf,
                                [g.to(x.device) for g in grads])
    assert dx.dtype == x.dtype and dx.shape == x.shape
    n = n or c
    ref, tol = lp_formula(x.cpu(), labels.cpu(), n, k, grads)
    assert torch.equal(out[3].cpu(), ref[3])
    for i, name in enumerate(("logp", "entropy", "top_logp")):
        close(out[i], ref[i], tol[i], name)
    assert not dx[:, n:].float().any()
    close(dx[:, :n], ref[4],
          tol[4] + half(x.dtype) * ref[4].abs()
          + torch.finfo(x.dtype).tiny, "dlogits")
    return [*out, dx]


def lp_inputs(rows, c, dtype, device, n=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = (3 * torch.randn(rows, c, generator=g)).to(dtype)
    labels = torch.randint(0, n or c, (rows,), generator=g)
    return x.to(device), labels.to(device)


@pytest.mark.parametrize("rows,c,n,k", [(5, 7, None, 3), (4, 16, 10, 10),
                                        (1, 1, None, 1), (0, 3, None, 2),
                                        (3, 5, None, 0)])
def test_label_logprobs_cpu(rows, c, n, k):
    for dtype in TYPES:
        lp_check(*lp_inputs(rows, c, dtype, "cpu", n), n=n, k=k)


def test_label_logprobs_gradient_against_differences():
    x, _ = lp_inputs(5, 8, torch.float32, "cpu")
    x = x.double()
    x[1, 2:4] = float("-inf")
    labels = torch.tensor([0, 5, -1, 6, 3])
    free = x.clone().requires_grad_(True)
    for r in range(5):            # differences need finite entries
        if torch.isfinite(x[r]).all():
            assert torch.autograd.gradcheck(
                lambda t: OF.label_logprobs(t, labels[r:r + 1], n_classes=7,
                                            top=3)[:3],
                (free[r:r + 1].detach().requires_grad_(True),))


LP_SHAPES = [(1, 1, None, 1), (3, 2, None, 2), (9, 10, None, 5),
             (128, 1008, 1000, 5), (5, 511, None, 32), (6, 513, 512, 7),
             (4, 1025, None, 3), (3, 2049, 2040, 20), (2, 9001, None, 8),
             (70, 20000, 19999, 4), (1, 131073, None, 32),
             (2, 300007, 300001, 9), (3, 8192, None, 0),
             (600, 17003, 16999, 4), (9, 1500, None, 6), (5, 2500, 2499, 6),
             (1100, 5001, None, 3)]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,c,n,k", LP_SHAPES)
def test_label_logprobs_gpu(rows, c, n, k, dtype):
    x, labels = lp_inputs(rows, c, dtype, dev(), n)
    if n is not None:
        x[:, n:] = float("nan")             # never read
    lp_check(x, labels, n=n, k=k)


def lp_hard(c, dtype, device):
    """Rows of masks, ties and single classes."""
    inf = float("inf")
    x, _ = lp_inputs(12, c, dtype, "cpu")
    labels = torch.arange(12) % c
    x[0] = -inf                                   # nothing left
    labels[1] = -1                                # no class given
    x[2, 1:] = -inf                               # one class left
    labels[2] = 0
    x[3, ::2] = -inf                              # the given one masked
    labels[3] = 0
    x[4] = 1.5                                    # all alike
    x[5] = torch.randint(-2, 2, (c,)).to(dtype)   # many alike
    x[6, c // 2:] = -inf
    x[7, :c // 2] = -inf
    x[8] = torch.where(torch.arange(c) % 3 == 0, 0.0, -0.0)  # signed zeros
    x[9] = torch.finfo(dtype).min                 # a mask of that type
    x[9, c - 1] = 0.0
    x[10] = -inf                                  # nothing left, no class
    labels[10] = -100
    x[11] = x[11] * 30                            # one stands out
    return x.to(device), labels.to(device)


@pytest.mark.parametrize("dtype", TYPES)
def test_label_logprobs_masks_and_ties_cpu(dtype):
    torch.manual_seed(0)
    lp_check(*lp_hard(40, dtype, "cpu"), k=9)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("c", [40, 700, 5000, 40001])
def test_label_logprobs_masks_and_ties_gpu(c, dtype):
    torch.manual_seed(0)
    for k in (0, 1, 9, 32):
        lp_check(*lp_hard(c, dtype, dev()), k=k)


def lp_nan_check(device):
    inf, nan = float("inf"), float("nan")
    for c in (12, 3000, 70000):
        x, labels = lp_inputs(6, c, torch.float32, device)
        x[0, 3] = nan
        x[1, 4] = inf
        x[2] = -inf
        x[2, 5] = nan
        labels[3] = c                      # behind the classes
        labels[4] = 2 ** 40
        x = x.requires_grad_(True)
        out = OF.label_logprobs(x, labels, top=4)
        (dx,) = torch.autograd.grad((out[0].sum() + out[1].sum(),), x)
        assert torch.isnan(out[0][:5]).all()
        assert torch.isnan(out[1][:3]).all()
        assert torch.isfinite(out[1][3:]).all()
        assert torch.isfinite(out[0][5])
        assert torch.isnan(dx[3:5]).all() and torch.isfinite(dx[5]).all()
        # a NaN ranks first, an infinity before what is finite
        assert out[3][0, 0] == 3 and out[3][1, 0] == 4
        assert out[3][2].tolist() == [5, 0, 1, 2]
        assert torch.isfinite(out[2][3:]).all()


def test_label_logprobs_nan_and_bad_labels_cpu():
    lp_nan_check("cpu")


@gpu
def test_label_logprobs_nan_and_bad_labels_gpu():
    lp_nan_check(dev())


def lp_nan_first_check(device, dtype):
    """NaN in the first class, in all and in the first few of them: the
    alternatives are those of a stable sort, whatever their number."""
    nan = float("nan")
    for c, k in ((1, 1), (10, 10), (32, 32), (40, 7), (3000, 5), (9001, 32),
                 (70000, 8)):
        x, labels = lp_inputs(5, c, dtype, device)
        x[0, 0] = nan
        x[1] = nan
        x[2, :3] = nan
        x[3, ::2] = nan
        x[3, 1::2] = float("inf")
        out = OF.label_logprobs(x, labels, top=k)
        want = torch.sort(x.float().cpu(), dim=1, descending=True,
                          stable=True).indices[:, :k]
        assert torch.equal(out[3].cpu(), want), (c, k)
        for t in out[:3]:
            assert torch.isnan(t[:4]).all() and torch.isfinite(t[4]).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_label_logprobs_nan_first_cpu(dtype):
    lp_nan_first_check("cpu", dtype)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_label_logprobs_nan_first_gpu(dtype):
    lp_nan_first_check(dev(), dtype)


@gpu
@pytest.mark.parametrize("c", [5, 700, 5000, 40001])
def test_label_logprobs_gpu_large_maxima(c):
    """Maxima whose product with log2 e loses from a part of 1 to some 128 in
    rounding, on either side (fp32's smallest normal power is 2^-126)."""
    peaks = [1e5, 1.2e7, 3e7, -3e7, 4e8, 2000019456.0, 2000027264.0,
             2147523840.0, -2000003840.0, -2000011648.0, 1.7e10, 3e38]
    g = torch.Generator().manual_seed(2)
    x = torch.tensor(peaks)[:, None].repeat(1, c)
    steps = torch.randint(0, 4, x.shape, generator=g) * 2.0 ** -23
    x = x - x.abs() * steps
    x[:, 3] = torch.tensor(peaks)
    x[::2, 1] = -math.inf
    labels = torch.full((len(peaks),), 3)
    grads = lp_grads(len(peaks), 3)
    leaf = x.to(dev()).requires_grad_(True)
    out = OF.label_logprobs(leaf, labels.to(dev()), top=3)
    (dx,) = torch.autograd.grad(out[:3], leaf, [t.to(dev()) for t in grads])
    # a logarithm of some hundred classes is below half a step of 3e38 in 64
    # bits, too: the formula takes what the rows are below their maxima,
    # which is exact and gives the same probabilities
    ref, tol = lp_formula(x.double() - x[:, 3:4].double(), labels, c, 3,
                          grads)
    assert torch.equal(out[3].cpu(), ref[3])
    for i, name in enumerate(("logp", "entropy", "top_logp")):
        close(out[i], ref[i], tol[i], name)
    close(dx, ref[4], tol[4] + U * ref[4].abs(), "dlogits")


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_label_logprobs_gpu_strides(dtype):
    x, labels = lp_inputs(9, 600, dtype, dev(), n=250)
    lp_check(x[:, 5:305], labels, n=300, k=4)
    lp_check(x[::2, 1:252], labels[::2], k=4)
    lp_check(x.t().contiguous().t()[:, :251], labels, k=4)
    lp_check(x[:1, :260].expand(9, -1), labels, k=4)


@gpu
def test_label_logprobs_gpu_single_gradients():
    """Each of the three outputs alone, the others without a gradient."""
    x, labels = lp_inputs(7, 900, torch.float32, dev())
    ref = x.double().cpu().requires_grad_(True)
    leaf = x.requires_grad_(True)
    for pick in range(3):
        w = torch.randn(7, 5) if pick == 2 else torch.randn(7)
        (got,) = torch.autograd.grad(
            OF.label_logprobs(leaf, labels, top=5)[pick], leaf, w.to(dev()))
        (want,) = torch.autograd.grad(
            OF.label_logprobs(ref, labels.cpu(), top=5)[pick], ref,
            w.double())
        # entries are sums of two terms no larger than the weights
        close(got, want, DEPTH * U * 8 * float(w.abs().sum(-1).max()
                                               if pick == 2
                                               else w.abs().max()))


@gpu
def test_label_logprobs_gpu_agrees_with_the_fused_loss():
    """-mean(logp) is softmax_xent's loss, the first alternative its
    prediction."""
    x, labels = lp_inputs(64, 1008, torch.bfloat16, dev(), n=1000)
    loss, _, err = OF.softmax_xent_err(x, labels, 1000)
    logp, _, _, idx = OF.label_logprobs(x, labels, n_classes=1000, top=1)
    # __logf and __expf there: a few fp32 steps on values below 32
    assert abs(float(loss + logp.mean())) < 32 * DEPTH * U
    assert float(err) == pytest.approx(
        float((idx[:, 0] != labels).float().mean()))


@gpu
def test_label_logprobs_gpu_most_classes():
    for dtype, most in ((torch.float32, 2 ** 21), (torch.bfloat16, 2 ** 22)):
        x = torch.zeros(1, most + 1, dtype=dtype, device=dev())
        x[0, most - 1] = 20.0
        labels = torch.full((1,), most - 1, device=dev())
        logp, _, _, idx = OF.label_logprobs(x, labels, n_classes=most,
                                            top=3)
        want = -math.log1p((most - 1) * math.exp(-20.0))
        # sums of 2^22 equal terms: DEPTH roundings of the sum, on its
        # logarithm, and of the logit
        assert abs(float(logp) - want) < DEPTH * U + 40 * U
        assert idx[0].tolist() == [most - 1, 0, 1]
        with pytest.raises(RuntimeError):
            OF.label_logprobs(x, labels)


@gpu
def test_label_logprobs_gpu_more_rows_than_a_launch():
    rows, tail = 2 ** 23 + 9, 100
    x = torch.randn(rows, 10, device=dev()).bfloat16()
    labels = torch.arange(rows, device=dev()) % 10
    whole = x.requires_grad_(True)
    part = x.detach()[-tail:].clone().requires_grad_(True)
    got = OF.label_logprobs(whole, labels, top=2)
    want = OF.label_logprobs(part, labels[-tail:], top=2)
    for a, b in zip(got, want):
        assert torch.equal(a[-tail:], b)
    (dx,) = torch.autograd.grad(got[0].sum() + got[2].sum(), whole)
    (dw,) = torch.autograd.grad(want[0].sum() + want[2].sum(), part)
    assert torch.equal(dx[-tail:], dw)


def test_label_logprobs_refusals():
    x, labels = lp_inputs(4, 9, torch.float32, "cpu")
    with pytest.raises(TypeError):
        OF.label_logprobs(x.long(), labels)
    with pytest.raises(TypeError):
        OF.label_logprobs(x, labels.int())
    for bad in (labels[:3], labels[None]):
        with pytest.raises(ValueError):
            OF.label_logprobs(x, bad)
    for bad in (x[0], x[None], x[:, :0]):
        with pytest.raises(ValueError):
            OF.label_logprobs(bad, labels)
    for n in (0, 10, -1, 3.0):
        with pytest.raises(ValueError):
            OF.label_logprobs(x, labels, n_classes=n)
    for k in (-1, 10, 2.0, True):
        with pytest.raises(ValueError):
            OF.label_logprobs(x, labels, top=k)
    with pytest.raises(ValueError):
        OF.label_logprobs(x, labels, n_classes=3, top=4)
    with pytest.raises(ValueError):
        OF.label_logprobs(torch.zeros(2, 99), torch.zeros(2).long(), top=33)
    with pytest.raises(ValueError):
        OF.label_logprobs(x, labels.to("meta"))


# ---------------------------------------------------------------------------
# orthogonalising, the momentum update
# ---------------------------------------------------------------------------

def ns_formula(x, steps=5):
    """By singular values: the iteration acts on them alone."""
    x = x.double().cpu()
    norm = torch.linalg.vector_norm(x, dim=(-2, -1), keepdim=True)
    u, s, vh = torch.linalg.svd(x / (norm + 1e-7), full_matrices=False)
    a, b, c = OF.NS_QUINTIC
    for _ in range(steps):
        s = a * s + b * s ** 3 + c * s ** 5
    return (u * s[..., None, :]) @ vh


def off(got, ref):
    """Distance relative to the reference, in the Frobenius norm."""
    got, ref = got.detach().double().cpu(), ref.double().cpu()
    assert got.shape == ref.shape
    return float((got - ref).norm() / ref.norm().clamp_min(1e-300))


# A product of fp32-like operands is off by about e = 2^-20 of its
# factors' norms (22-bit operands, three of them, and the additions).
# With singular values up to 1.21, B = aI + bA + cAA is off by
# (|b| 1.46 + 2 c 2.14) e = 16 e, and X <- BX by (16 + 3.5) e; five steps
# of that, at slopes around 1 where the singular values gather, are 100 e.
NS_TOL = 100 * 2.0 ** -20


def ns_inputs(shape, dtype, device, seed=0, scale=1e-3):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(*shape, generator=g)).to(dtype).to(device)


@pytest.mark.parametrize("shape", [(1, 1), (4, 9), (9, 4), (3, 5, 6)],
                         ids=str)
def test_orthogonalize_cpu(shape):
    for dtype in TYPES:
        x = ns_inputs(shape, dtype, "cpu")
        y = OF.orthogonalize(x)
        assert y.dtype == dtype and y.is_contiguous()
        assert off(y, ns_formula(x)) < NS_TOL + half(dtype)


NS_SHAPES = [(1, 1), (1, 300), (300, 1), (2, 3), (16, 16), (63, 65),
             (64, 64), (65, 63), (64, 576), (200, 129), (10, 256),
             (2304, 256), (500, 700), (3, 100, 70), (2, 64, 800),
             (5, 1, 7)]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", NS_SHAPES, ids=str)
def test_orthogonalize_gpu(shape, dtype):
    # fp16 has no numbers for gradients of 1e-6
    x = ns_inputs(shape, dtype, dev(), scale=0.05)
    y = OF.orthogonalize(x)
    assert y.dtype == dtype and y.shape == x.shape
    assert off(y, ns_formula(x)) < NS_TOL + half(dtype)


@gpu
@pytest.mark.parametrize("shape", [(90, 150), (40, 330)], ids=str)
@pytest.mark.parametrize("steps", [1, 2, 3, 4, 8])
def test_orthogonalize_gpu_steps(steps, shape):
    x = ns_inputs(shape, torch.float32, dev())
    assert off(OF.orthogonalize(x, steps),
               ns_formula(x, steps)) < NS_TOL * max(1, steps / 5)


def ns_recurrence(x, steps=5):
    """The definition in 64 bits, where a singular value decomposition
    would take minutes."""
    x = x.double()
    x = x / (torch.linalg.vector_norm(x) + 1e-7)
    a, b, c = OF.NS_QUINTIC
    for _ in range(steps):
        g = x @ x.t()
        x = a * x + (b * g + c * g @ g) @ x
    return x


# One shape for each way through the kernels: k cut into runs and not,
# tiles of 64 with one, two and more blocks a compute unit, of 128 and 256,
# two steps at a time and one, the padding of m and n within a tile; few
# rows in many groups of columns.
@gpu
@pytest.mark.parametrize("shape,steps", [
    ((70, 5000), 5), ((700, 1100), 5), ((1300, 4650), 5), ((1300, 4650), 4),
    ((2500, 2500), 5), ((2050, 8200), 5), ((4097, 4100), 3),
    ((33, 40003), 5), ((600, 4700), 5), ((1030, 1100), 5),
    ((1000, 8000), 5), ((1800, 4500), 5), ((2050, 12000), 5)], ids=str)
def test_orthogonalize_gpu_large(shape, steps):
    x = ns_inputs(shape, torch.float32, dev())
    want = ns_recurrence(x, steps)
    assert off(OF.orthogonalize(x, steps), want) < NS_TOL
    tall = x.t().contiguous()
    assert off(OF.orthogonalize(tall, steps).t(), want) < NS_TOL


@gpu
@pytest.mark.parametrize("shape", [(5, 100, 300), (3, 1000, 2100),
                                   (7, 130, 65), (2, 2100, 1000),
                                   (2, 1200, 4700), (5, 1100, 2400)],
                         ids=str)
def test_orthogonalize_gpu_batches(shape):
    x = ns_inputs(shape, torch.float32, dev())
    y = OF.orthogonalize(x)
    for i in range(shape[0]):
        m = x[i] if shape[1] <= shape[2] else x[i].t()
        want = ns_recurrence(m, 5)
        assert off(y[i], want if shape[1] <= shape[2]
                   else want.t()) < NS_TOL


@gpu
def test_orthogonalize_gpu_same_bits_again():
    for shape in ((64, 576), (300, 2000), (1300, 4650)):
        x = ns_inputs(shape, torch.float32, dev())
        assert torch.equal(OF.orthogonalize(x), OF.orthogonalize(x))


@gpu
@pytest.mark.parametrize("shape", [(96, 400), (256, 256)], ids=str)
def test_orthogonalize_gpu_weak_directions(shape):
    """One strong direction over noise of a ten-thousandth: the noise is
    amplified up to 485 times, and with it what the operands lose.  An
    operand of 22 bits is off by 2^-23 of its entries; 485 times that,
    over two operands and a norm of the result of at least that of the
    strong direction (0.7), is 2^-13; operands of 8 or 11 bits alone
    would miss it by 2^9 and more."""
    g = torch.Generator().manual_seed(3)
    x = torch.outer(torch.randn(shape[0], generator=g),
                    torch.randn(shape[1], generator=g))
    x = (x + 1e-4 * torch.randn(*shape, generator=g)).to(dev())
    assert off(OF.orthogonalize(x), ns_formula(x)) < 2.0 ** -13


def ns_gradient(shape, seed):
    """Up to 16 strong directions of falling strength over noise."""
    g = torch.Generator().manual_seed(seed)
    rank = max(1, min(16, min(shape) // 4))
    left = torch.randn(shape[0], rank, generator=g)
    left *= torch.logspace(0, -1, rank)
    strong = left @ torch.randn(rank, shape[1], generator=g)
    return (1e-3 * (strong + 0.5 * torch.randn(*shape, generator=g))).to(
        dev())


def ns_error_check(mats, got):
    """Distances from 64 bits, of the kernels and of plain fp32 products.
    Operands of 22 bits are rounded at twice to four times fp32's step, which
    shows where sums are short: twice plain fp32's error is allowed.  In
    long sums the additions' roundings are most of it, and both have these:
    from 128 rows on no more than plain fp32's is."""
    want = [ns_recurrence(m) for m in mats]
    plain = [OF.orthogonalize_ref(m) for m in mats]
    ours = sum(off(a, b) for a, b in zip(got, want))
    fp32 = sum(off(a, b) for a, b in zip(plain, want))
    few = min(mats[0].shape) < 128
    assert ours < (2.0 if few else 1.0) * fp32, (ours, fp32)


@gpu
@pytest.mark.parametrize("shape", [
    (32, 2000), (48, 192), (64, 256), (65, 130), (65, 576), (128, 256),
    (128, 1152), (256, 512), (350, 700), (512, 2000), (800, 1600),
    (2000, 4000), (2500, 2500), (4096, 4096), (4096, 9216)], ids=str)
def test_orthogonalize_gpu_errors_of_float32(shape):
    mats = [ns_gradient(shape, s) for s in range(6 if shape[0] < 512 else 1)]
    ns_error_check(mats, [OF.orthogonalize(m) for m in mats])


@gpu
def test_muon_update_gpu_errors_in_a_list():
    """Short matrices among long ones: with nothing kept of the weight, the
    momentum all new and a rate of 1 a weight is its orthogonalised gradient."""
    shapes = [(16, 27), (128, 128), (64, 64), (128, 1152), (256, 2304),
              (256, 256), (512, 4608), (65, 130)]
    runs = []
    for seed in range(4):
        mats = [ns_gradient(s, seed * 10 + i) for i, s in enumerate(shapes)]
        ws = [torch.zeros_like(m) for m in mats]
        vs = [torch.zeros_like(m) for m in mats]
        many = len(mats)
        OF.muon_update(ws, [-m for m in mats], vs, [None] * many,
                       [1.0] * many, [0.0] * many, 0.9, [1.0] * many)
        runs.append((mats, ws))
    for i in range(len(shapes)):
        ns_error_check([m[i] for m, _ in runs], [w[i] for _, w in runs])


@gpu
@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e15, 1e30])
def test_orthogonalize_gpu_magnitudes(scale):
    x = ns_inputs((70, 90), torch.float32, dev(), scale=scale)
    assert off(OF.orthogonalize(x), ns_formula(x)) < NS_TOL


@gpu
@pytest.mark.parametrize("shape", [(40, 100), (64, 9000), (70, 150),
                                   (600, 2000), (1300, 8000)], ids=str)
@pytest.mark.parametrize("scale,steps", [
    (1e-12, 3), (1e-12, 10), (1e-16, 14), (1e-20, 12), (1e-20, 20),
    (1e-20, 27), (1e-30, 1), (1e-30, 40), (1e-30, 44), (3e-38, 2),
    (3e-38, 60)])
def test_orthogonalize_gpu_small_norms_and_many_steps(scale, steps, shape):
    """Norms far below 1e-7 leave X as far below 1, which takes a step for
    each factor of 3.4445 to grow: on the way there and a few steps after
    (singular values that have grown go to and fro between 0.7 and 1.2, and
    tens of such steps would make any rounding large)."""
    x = ns_inputs(shape, torch.float32, dev(), scale=scale)
    want = ns_recurrence(x, steps)
    assert 0 < float(want.norm()) < 1.3 * math.sqrt(shape[0])
    assert off(OF.orthogonalize(x, steps), want) < NS_TOL * max(1, steps / 5)


@gpu
def test_orthogonalize_gpu_small_norms_in_a_batch():
    scales = (1e-15, 1e-18, 1e-20, 0.0, 1e-30)
    for shape in ((30, 50), (80, 90)):
        x = torch.stack([ns_inputs(shape, torch.float32, dev(), scale=s,
                                   seed=i) for i, s in enumerate(scales)])
        y = OF.orthogonalize(x, 20)
        for i, s in enumerate(scales):
            if s:
                assert off(y[i], ns_recurrence(x[i], 20)) < NS_TOL * 20 / 5
            else:
                assert not y[i].any()


@gpu
def test_orthogonalize_gpu_zero_nan_empty():
    x = torch.zeros(3, 40, 50, device=dev())
    x[1] = torch.randn(40, 50, device=dev())
    x[2, 7, 3] = float("nan")
    y = OF.orthogonalize(x)
    assert not y[0].any() and torch.isnan(y[2]).all()
    assert off(y[1], ns_formula(x[1])) < NS_TOL
    for shape in ((0, 3, 4), (0, 4), (4, 0)):
        assert OF.orthogonalize(torch.zeros(shape,
                                            device=dev())).shape == shape


@gpu
def test_orthogonalize_gpu_strides():
    x = ns_inputs((2, 60, 90), torch.float32, dev())
    for t in (x.transpose(1, 2), x[:, ::2, 1:80], x.transpose(0, 1),
              x[:1].expand(3, -1, -1)):
        y = OF.orthogonalize(t)
        assert y.is_contiguous()
        assert off(y, ns_formula(t)) < NS_TOL


def muon_inputs(shapes, device, seed=0):
    g = torch.Generator().manual_seed(seed)

    def some(scale):
        return [(scale * torch.randn(*s, generator=g)).to(device)
                for s in shapes]
    ws, gs, vs = some(1.0), some(1e-3), some(4e-3)
    return ws, gs, vs, [w.to(torch.bfloat16) for w in ws]


def muon_check(shapes, device, phase=0, copies=True):
    ws, gs, vs, outs = muon_inputs(shapes, device)
    if not copies:
        outs = [o if i % 2 else None for i, o in enumerate(outs)]
    many = len(ws)
    lrs = [0.02 + 0.01 * i for i in range(many)]
    wds = [0.1 * (i % 3) for i in range(many)]
    scales = [1.0 + i for i in range(many)]
    old = [[t.double().cpu() for t in part] for part in (ws, gs, vs)]
    given = gs if phase != 2 else [None] * many        # not read
    OF.muon_update(ws, given, vs, outs, lrs, wds, 0.9, scales, phase)
    for i in range(many):
        w, g, v = (part[i] for part in old)
        if phase != 2:
            close(vs[i], 0.9 * v - g, 3 * U * (v.abs() + g.abs()), "v")
            v = vs[i].double().cpu()      # what was stored goes on
        else:
            assert torch.equal(vs[i].double().cpu(), v)
        if phase == 1:
            assert torch.equal(ws[i].double().cpu(), w)
            continue
        o = ns_formula(v)
        step = lrs[i] * scales[i]
        want = (1 - lrs[i] * wds[i]) * w + step * o
        diff = ws[i].double().cpu() - want
        size = float((3 * U * (w.abs() + want.abs())).norm())
        assert float(diff.norm()) <= size + step * NS_TOL * float(o.norm())
        if outs[i] is not None:
            assert torch.equal(outs[i], ws[i].to(torch.bfloat16))


@pytest.mark.parametrize("phase", [0, 1, 2])
def test_muon_update_cpu(phase):
    muon_check([(3, 4), (6, 2), (2, 5, 3)], "cpu", phase, copies=False)


@gpu
@pytest.mark.parametrize("phase", [0, 1, 2])
def test_muon_update_gpu(phase):
    muon_check([(16, 27), (64, 576), (10, 256), (256, 10), (1, 1),
                (3, 48, 70), (130, 130)], dev(), phase)


@gpu
@pytest.mark.parametrize("shapes", [
    [(16, 27), (64, 576), (10, 256), (2, 3, 50)],      # few rows alone
    [(16, 27), (128, 700), (1300, 4700), (64, 64)],
    [(16, 27), (128, 700), (1800, 4500), (64, 64)]],
                         ids=["few", "mixed", "large"])
def test_muon_update_gpu_kinds(shapes):
    """Lists whose matrices take the same kernels and several kinds."""
    muon_check([s for s in shapes if s[0] < 1000], dev())
    if len(shapes[2]) == 2 and shapes[2][0] > 1000:
        ws, gs, vs, outs = muon_inputs(shapes, dev())
        want = [(w.double() * 0.998, 0.9 * v.double() - g.double())
                for w, g, v in zip(ws, gs, vs)]
        OF.muon_update(ws, gs, vs, outs, [0.02] * 4, [0.1] * 4, 0.9,
                       [5.0] * 4)
        for w, v, (keep, vel) in zip(ws, vs, want):
            close(v, vel, 3 * U * (vel.abs() + 0.02), "v")
            o = ns_recurrence(vel if vel.shape[0] <= vel.shape[1]
                              else vel.t())
            diff = w.double() - (keep + 0.1 * o)
            assert float(diff.norm()) <= (
                6 * U * float(keep.norm()) + 0.1 * NS_TOL * float(o.norm()))


@gpu
def test_muon_update_gpu_long_list_without_copies():
    muon_check([(3 + i, 70 - 2 * i) for i in range(30)], dev(),
               copies=False)


def muon_refusals(device):
    def call(phase=0, steps=5, **change):
        parts = dict(zip(("ws", "gs", "vs", "outs"),
                         muon_inputs([(4, 6), (3, 5)], device)))
        kept = [t.clone() for t in parts["ws"]]
        lists = {"lrs": [0.1, 0.1], "wds": [0.0, 0.0],
                 "scales": [1.0, 1.0]}
        for k, f in change.items():
            for d in (parts, lists):
                if k in d:
                    d[k] = f(d[k])
        error = None
        try:
            OF.muon_update(parts["ws"], parts["gs"], parts["vs"],
                           parts["outs"], lists["lrs"], lists["wds"], 0.9,
                           lists["scales"], phase, steps)
        except (TypeError, ValueError) as e:
            error = e
        if not any(k == "ws" for k in change):
            assert all(torch.equal(a, b)
                       for a, b in zip(kept, parts["ws"]))
        return error

    for k in ("gs", "vs", "outs", "lrs", "wds", "scales"):
        assert isinstance(call(**{k: lambda v: v[:1]}), ValueError), k
    for k in ("ws", "gs", "vs"):
        assert isinstance(call(**{k: lambda v: [v[0], v[1].double()]}),
                          TypeError)
        assert isinstance(call(**{k: lambda v: [v[0], v[1].t()]}),
                          ValueError)
        assert isinstance(call(**{k: lambda v: [v[0], v[1][:2]]}),
                          ValueError)
    assert isinstance(call(outs=lambda v: [v[0], v[1].float()]), TypeError)
    assert isinstance(call(outs=lambda v: [v[0], v[1][:1]]), ValueError)
    same = lambda v: [v[0], v[0].view(4, 6)]          # noqa: E731
    for k in ("ws", "vs", "outs"):
        every = {j: (same if j == k else lambda v: [
            v[0], v[0].clone()]) for j in ("ws", "gs", "vs", "outs")}
        assert isinstance(call(**every), ValueError), k
    assert isinstance(call(phase=3), ValueError)
    for steps in (0, 65, 2.0):
        assert isinstance(call(steps=steps), ValueError)


def muon_shared_memory(device):
    """Overlaps are refused, whatever their start, and nothing is written;
    neighbours in one buffer and a gradient for two weights are fine."""
    def call(change):
        flat = torch.randn(400, device=device)
        cut = lambda at, rows=4: flat[at:at + rows * 5].view(  # noqa: E731
            rows, 5)
        parts = {"ws": [cut(0), cut(20)], "gs": [cut(40), cut(60)],
                 "vs": [cut(80), cut(100)],
                 "outs": [cut(120, 2).view(torch.bfloat16).view(4, 5), None]}
        change(parts, cut)
        kept = flat.clone()
        try:
            OF.muon_update(parts["ws"], parts["gs"], parts["vs"],
                           parts["outs"], [0.1] * 2, [0.0] * 2, 0.9,
                           [1.0] * 2)
        except ValueError:
            assert torch.equal(flat, kept)
            return False
        return True

    def put(name, i, at):
        return lambda parts, cut: parts[name].__setitem__(i, cut(at))

    assert call(lambda parts, cut: None)
    assert call(put("gs", 1, 40))                 # one gradient for two
    for name, i, at in (("ws", 1, 0), ("ws", 1, 5), ("ws", 0, 15),
                        ("vs", 0, 101), ("vs", 1, 15), ("gs", 0, 0),
                        ("gs", 1, 79), ("gs", 0, 99), ("gs", 1, 125),
                        ("ws", 0, 110), ("vs", 0, 121)):
        assert not call(put(name, i, at)), (name, i, at)


def test_muon_update_shared_memory_cpu():
    muon_shared_memory("cpu")


@gpu
def test_muon_update_shared_memory_gpu():
    muon_shared_memory(dev())


def test_muon_update_refusals_cpu():
    muon_refusals("cpu")
    OF.muon_update([], [], [], [], [], [], 0.9, [])


@gpu
def test_muon_update_refusals_gpu():
    muon_refusals(dev())
    ws, gs, vs, outs = muon_inputs([(4, 6)], dev())
    with pytest.raises(ValueError):
        OF.muon_update(ws, [gs[0].cpu()], vs, outs, [0.1], [0.0], 0.9,
                       [1.0])


def test_orthogonalize_refusals():
    x = torch.ones(3, 4)
    for bad in (x[0], x[None, None]):
        with pytest.raises(ValueError):
            OF.orthogonalize(bad)
    with pytest.raises(TypeError):
        OF.orthogonalize(x.int())
    for steps in (0, 65, 2.5, True):
        with pytest.raises(ValueError):
            OF.orthogonalize(x, steps)


# ---------------------------------------------------------------------------
# the optimizer, the layer, and all of them together
# ---------------------------------------------------------------------------

def test_muon_optimizer_phases_and_rest_cpu():
    """step() is phase1() then phase2(); matrices are orthogonalised,
    other parameters take the SGD step."""
    from theanompi_amd.lib.opt import Muon, ParamRec, SGDMomentum

    def recs():
        torch.manual_seed(0)
        w = torch.nn.Parameter(torch.randn(2, 3, 5))
        b = torch.nn.Parameter(torch.randn(4))
        w.grad, b.grad = torch.randn(2, 3, 5), torch.randn(4)
        return [ParamRec(w, "W", matrix=(2, 3, 5)), ParamRec(b, "b")]

    whole, split, sgd = recs(), recs(), recs()
    kw = dict(lr=0.1, momentum=0.9, weight_decay=0.01)
    a, b = Muon(whole, **kw), Muon(split, **kw)
    for _ in range(2):
        a.step()
        b.phase1()
        b.phase2()
    for x, y in zip(whole, split):
        assert torch.equal(x.master.data, y.master.data)
    plain = SGDMomentum([sgd[1]], **kw)
    plain.step()
    plain.step()
    assert torch.equal(sgd[1].master.data, whole[1].master.data)
    # an update's root mean square is lr * rms, within the band that the
    # singular values end in
    before = whole[0].master.data.clone()
    a.step()
    delta = whole[0].master.data - (1 - 0.1 * 0.01) * before
    rms = float(delta.square().mean().sqrt())
    assert 0.5 * 0.1 * 0.2 < rms < 1.3 * 0.1 * 0.2


def muon_recs_without_gradients(device):
    """A trained matrix, a frozen one, one that got a single gradient, and
    their optimizer under each way to step."""
    from theanompi_amd.lib.opt import Muon, ParamRec
    after = []
    for way in ("step", "phases", "persistent"):
        g = torch.Generator().manual_seed(0)
        ps = [torch.nn.Parameter(torch.randn(4, 6, generator=g).to(device))
              for _ in range(3)]
        ps[1].requires_grad_(False)
        recs = [ParamRec(p, matrix=(1, 4, 6)) for p in ps]
        opt = Muon(recs, lr=0.1, momentum=0.9, weight_decay=0.01)
        if way == "persistent":
            opt.make_persistent()
        start = [p.detach().clone() for p in ps]
        once = None
        for it in range(10):
            opt.zero_grad()
            grad = torch.randn(4, 6, generator=g).to(device)
            if way == "persistent":
                ps[0].grad.copy_(grad)
            else:
                ps[0].grad = grad
                ps[2].grad = 1e-6 * grad if it == 0 else None
            if way == "phases":
                opt.phase1()
                opt.phase2()
            else:
                opt.step()
            if it == 0:
                once = ps[2].detach().clone()
        assert not torch.equal(ps[0], start[0])
        assert torch.equal(ps[1], start[1]), way
        if way != "persistent":
            assert not torch.equal(once, start[2])
            assert torch.equal(ps[2], once), way
            after.append([p.detach().clone() for p in ps])
    for a, b in zip(*after):
        assert torch.equal(a, b)


def test_muon_leaves_weights_without_a_gradient_cpu():
    muon_recs_without_gradients("cpu")


@gpu
def test_muon_leaves_weights_without_a_gradient_gpu():
    muon_recs_without_gradients(dev())


def test_muon_phase2_by_itself_cpu():
    """Without a first phase the gradients that are there decide."""
    from theanompi_amd.lib.opt import Muon, ParamRec
    ps = [torch.nn.Parameter(torch.ones(3, 4)) for _ in range(2)]
    recs = [ParamRec(p, matrix=(1, 3, 4)) for p in ps]
    for r in recs:
        r.vel.copy_(torch.eye(3, 4))
    opt = Muon(recs, lr=0.1)
    ps[0].grad = torch.zeros(3, 4)
    opt.phase2()
    assert not torch.equal(ps[0], torch.ones(3, 4))
    assert torch.equal(ps[1], torch.ones(3, 4))


def test_optimizer_by_name():
    from theanompi_amd.lib import opt
    from theanompi_amd.models.cifar10 import Cifar10_model
    with pytest.raises(ValueError):
        opt.build_optimizer("adam", [])
    m = Cifar10_model({"device": "cpu", "n_iters": 2, "batch_size": 4,
                       "verbose": False, "optimizer": "muon"})
    m.compile_iter_fns("cdd")
    assert type(m.opt) is opt.Muon
    before = [p.detach().clone() for p in m.params]
    m.train_iter(0)
    m.apply_update()
    assert all(not torch.equal(a, b) for a, b in zip(before, m.params))
    m = Cifar10_model({"device": "cpu", "n_iters": 2, "batch_size": 4,
                       "verbose": False})
    m.compile_iter_fns("cdd")
    assert type(m.opt) is opt.SGDMomentum


@pytest.mark.parametrize("optimizer", ["sgd", "muon"])
def test_wrapped_module_with_an_empty_parameter(optimizer):
    from theanompi_amd.models.module_adapter import wrap_module

    class Net(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.none = torch.nn.Parameter(torch.zeros(0, 5))
            self.fc = torch.nn.Linear(3 * 16 * 16, 10)

        def forward(self, x):
            return self.fc(x.flatten(1)) + self.none.sum()

    model = wrap_module(Net, batch_size=4, n_classes=10, image_hw=16)
    m = model({"device": "cpu", "verbose": False, "n_iters": 1,
               "optimizer": optimizer})
    m.compile_iter_fns("cdd")
    before = m.module.fc.weight.detach().clone()
    m.train_iter(0)
    m.apply_update()
    assert not torch.equal(before, m.module.fc.weight)


def test_layernorm_layer_cpu():
    from theanompi_amd.models import layers as L
    ln = L.LayerNorm(10)
    x = torch.randn(3, 10)
    assert off(ln(x), torch.nn.functional.layer_norm(x.double(),
                                                     (10,))) < 16 * U
    names = [n for n, _, _ in ln.logical_params()]
    assert names == ["gamma", "beta"]


@gpu
def test_muon_trains_a_model_gpu():
    """A convolutional network's step: padded weight entries stay 0, the
    working copies follow the masters, and every weight moves by about
    lr * rms (between half and 1.3 times: the singular values end between
    0.68 and 1.21, and merged or padded matrices have some at 0)."""
    from theanompi_amd.lib.opt import Muon
    from theanompi_amd.models.cifar10 import Cifar10_model
    for sync in ("cdd", "avg", "grad"):
        m = Cifar10_model({"device": "cuda:0", "n_iters": 2,
                           "batch_size": 16, "verbose": False,
                           "optimizer": "muon"})
        m.compile_iter_fns(sync)
        assert type(m.opt) is Muon
        before = [r.master.data.clone() for r in m.recs]
        m.train_iter(0)
        m.apply_update()
        for r, b in zip(m.recs, before):
            w = r.master.data
            assert torch.isfinite(w).all()
            if r.matrix is None:
                continue
            assert not w[b == 0].any()
            assert torch.equal(r.bf16_out, w.to(torch.bfloat16))
            lr, wd = m.opt.lr, m.opt.weight_decay
            step = (w - (1 - lr * wd) * b)[b != 0]
            rms = float(step.square().mean().sqrt()) / (lr * m.opt.rms)
            assert 0.3 < rms < 1.3, (sync, r.name, rms)


class _Head(torch.nn.Module):
    """Features -> layer norm -> classes."""

    def __init__(self, device, batch):
        super().__init__()
        from theanompi_amd.models import layers as L
        self.fc1 = L.Linear(48, 100, device=device, batch=batch)
        self.norm = L.LayerNorm(100, device=device)
        self.fc2 = L.Linear(100, 21, device=device, batch=batch)

    def forward(self, x):
        return self.fc2(OF.relu(self.norm(self.fc1(x))))


def _head_step(device, weights=None):
    """Loss, gradients and updated weights of one step, as logical
    parameters: mean of -logp, less a little entropy."""
    from theanompi_amd.lib.opt import Muon, ParamRec
    torch.manual_seed(0)
    m = _Head(str(device), 32)
    mods = [m.fc1, m.norm, m.fc2]
    if weights is not None:
        flat = iter(weights)
        for mod in mods:
            for _, _, put in mod.logical_params():
                put(next(flat).clone())
    start = [get().detach().clone().cpu() for mod in mods
             for _, get, _ in mod.logical_params()]
    recs = []
    for mod in mods:
        if mod is m.norm:
            recs += [ParamRec(mod.gamma), ParamRec(mod.beta)]
        else:
            matrix, span = mod.weight_matrix()
            recs += [ParamRec(mod.weight, matrix=matrix, span=span,
                              bf16_out=getattr(mod, "w_bf16", None)),
                     ParamRec(mod.bias)]
    opt = Muon(recs, lr=0.05, momentum=0.9)
    g = torch.Generator().manual_seed(7)
    x = torch.randn(32, 48, generator=g).to(torch.bfloat16)
    y = torch.randint(0, 21, (32,), generator=g).to(device)
    x = x.to(device) if device.type == "cuda" else x.float()
    logits = m(x)
    logp, entropy, _, _ = OF.label_logprobs(logits, y, n_classes=21)
    loss = -logp.mean() - 0.01 * entropy.mean()
    loss.backward()
    grads = [r.master.grad.detach().clone() for r in recs]
    spans = [r.span for r in recs]

    def logical():
        return [get().detach().clone().cpu() for mod in mods
                for _, get, _ in mod.logical_params()]
    keep = [r.master.data for r in recs]
    for r, gr in zip(recs, grads):
        r.master.data = gr
    glog = logical()
    for r, w in zip(recs, keep):
        r.master.data = w
    opt.step()
    return start, float(loss.detach()), glog, logical(), spans


@gpu
def test_head_trains_like_the_cpu():
    """Layer norm, log probabilities and the orthogonalised update in one
    step, against the same on the CPU in fp32.  Activations and weights
    are rounded to bf16 about eight times between input and gradient, by
    2^-9 each in the mean; four times their root mean square is allowed.
    The update has the gradient's error times the slope of the iteration
    at weak directions relative to its result, at most 3.5."""
    start, loss, grads, after, spans = _head_step(torch.device("cpu"))
    _, loss_g, grads_g, after_g, spans_g = _head_step(dev(), start)
    assert spans == spans_g
    tol = 4 * math.sqrt(8) * 2.0 ** -9
    assert abs(loss - loss_g) < tol * abs(loss)
    for a, b in zip(grads, grads_g):
        assert off(b, a) < tol
    for s, a, b, name in zip(start, after, after_g, "WbgbWb"):
        s = s.double()
        assert off(b.double() - s, a.double() - s) < (
            3.5 * tol if name == "W" else tol)


@gpu
def test_operators_replay_in_a_graph():
    """Captured once, replayed on new data with eager work in between:
    every replay is the eager result, bit for bit."""
    x, gamma, beta, dy = ln_inputs((300, 512), torch.bfloat16, dev())
    labels = torch.randint(0, 500, (300,), device=dev())
    w, gr, v, out = [t[0] for t in muon_inputs([(96, 160)], dev())]
    leaf = x.detach().clone().requires_grad_(True)
    gl = gamma.detach().clone().requires_grad_(True)

    def step():
        y = OF.layernorm(leaf, gl, beta)
        logp, ent, top, idx = OF.label_logprobs(y, labels, n_classes=500,
                                                top=6)
        grads = torch.autograd.grad((logp, ent, top), (leaf, gl),
                                    (dlogp, dlogp * 0.1, dtop))
        OF.muon_update([w], [gr], [v], [out], [0.02], [0.01], 0.9, [2.0])
        return [y.detach(), logp.detach(), ent.detach(), idx, *grads, w, v,
                out]

    dlogp = torch.randn(300, device=dev())
    dtop = torch.randn(300, 6, device=dev())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(4):
        new = ln_inputs((300, 512), torch.bfloat16, dev(), seed=seed)
        nw = muon_inputs([(96, 160)], dev(), seed=seed)

        def put():
            with torch.no_grad():
                leaf.copy_(new[0])
                for t, s in zip((w, gr, v, out), nw):
                    t.copy_(s[0])
        put()
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        put()
        graph.replay()
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(held, want)):
            assert torch.equal(a, b), (seed, i)


@gpu
def test_operators_on_another_stream():
    """Work queued on a side stream, results read there."""
    args = ln_inputs((200, 1000), torch.bfloat16, dev())
    labels = torch.randint(0, 1000, (200,), device=dev())
    m = ns_inputs((100, 300), torch.float32, dev())

    def all_of():
        y = OF.layernorm(*args[:3])
        return [y, *OF.label_logprobs(y, labels, top=5),
                OF.orthogonalize(m)]
    want = all_of()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = all_of()
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


# ---------------------------------------------------------------------------
# offsets that 32 bits do not hold: the last rows against a call on these
# ---------------------------------------------------------------------------

@gpu
def test_layernorm_gpu_long_offsets():
    rows, c, tail = 270000, 8192, 40
    x = torch.empty(rows, c, dtype=torch.bfloat16, device=dev()).normal_()
    dy = torch.empty_like(x).normal_()
    _, gamma, beta, _ = ln_inputs((1, c), torch.float32, dev())
    leaf, end = x.requires_grad_(True), x.detach()[-tail:].clone()
    y = OF.layernorm(leaf, gamma, beta)
    (dx,) = torch.autograd.grad(y, leaf, dy)
    end.requires_grad_(True)
    ye = OF.layernorm(end, gamma, beta)
    (de,) = torch.autograd.grad(ye, end, dy[-tail:])
    assert torch.equal(y[-tail:], ye) and torch.equal(dx[-tail:], de)


@gpu
def test_layernorm_gpu_most_channels():
    """More channels than one launch of the last sum has threads for.  A
    lane adds up c / 1024 values, and the sums of 1024 lanes are joined."""
    c = 2 ** 25 + 37
    x, gamma, beta, dy = ln_inputs((2, c), torch.float32, dev())
    leaves = [t.requires_grad_(True) for t in (x, gamma, beta)]
    y = OF.layernorm(*leaves)
    got = [y, *torch.autograd.grad(y, leaves, dy)]
    ref, _ = ln_formula(x.detach(), gamma.detach(), beta.detach(), dy, 1e-5,
                        c)
    depth = c // 1024 + 32
    xh = (ref[0] - beta.detach().double()) / gamma.detach().double()
    e = depth * U * (xh.abs() + float(x.detach().abs().max()))
    ga, d = gamma.detach().double().abs(), dy.double().abs()
    tols = [ga * e + 4 * U * (ref[0].abs() + beta.detach().abs()),
            d * ga * e + 4 * depth * U * (d * ga + 1 + xh.abs()),
            (d * e).sum(0) + 4 * U * ref[2].abs(), 4 * U * d.sum(0)]
    for a, r, t, name in zip(got, ref, tols, ("y", "dx", "dgamma", "dbeta")):
        close(a, r, t, name)
    del ref, tols, xh, e
    with pytest.raises(RuntimeError):
        OF.layernorm(torch.empty(1, 2 ** 28 + 1, dtype=torch.bfloat16,
                                 device=dev()),
                     *(torch.empty(2 ** 28 + 1, device=dev())
                       for _ in range(2)))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_far_apart_gpu(dtype):
    """Rows whose offsets 32 bits do not hold, against the formulas."""
    far = 2 ** 29 - 11                  # elements from row to row
    for c in (1000, 9001):
        buf = torch.empty(9 * far + c, dtype=dtype, device=dev())
        x = buf.as_strided((10, c), (far, 1))
        new = ln_inputs((10, c), dtype, dev())
        x.copy_(new[0])
        ln_check(x, *new[1:])
        lp_check(x, torch.arange(10, device=dev()) * 7, k=3)
        del x, buf


@gpu
def test_label_logprobs_gpu_long_offsets():
    rows, c, tail = 17000, 131072, 40
    x = torch.empty(rows, c, dtype=torch.float16, device=dev()).normal_()
    labels = torch.arange(rows, device=dev()) * 7
    # the last rows again, among as many rows, which are cut alike
    again = x.roll(tail, 0)
    out = []
    for leaf, lab in ((x, labels), (again, labels.roll(tail, 0))):
        leaf.requires_grad_(True)
        got = OF.label_logprobs(leaf, lab, top=3)
        (dx,) = torch.autograd.grad(got[0].sum() + got[1].sum()
                                    + got[2].sum(), leaf)
        rows_of = slice(-tail, None) if leaf is x else slice(0, tail)
        out.append([t[rows_of].clone() for t in (*got, dx)])
        del got, dx
    for a, b in zip(*out):
        assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("shape", [(3000, 900, 800), (36000, 60, 1000)],
                         ids=str)
def test_orthogonalize_gpu_long_offsets_of_a_batch(shape):
    x = torch.empty(shape, dtype=torch.bfloat16, device=dev()).normal_()
    y = OF.orthogonalize(x)
    for i in (0, shape[0] // 2, shape[0] - 1):
        assert off(y[i], ns_formula(x[i])) < NS_TOL + half(x.dtype)


@gpu
@pytest.mark.parametrize("shape", [(11000000, 200), (200, 11000000),
                                   (64, 16777215)], ids=str)
def test_orthogonalize_gpu_long_offsets_of_a_matrix(shape):
    x = torch.empty(shape, device=dev()).normal_()
    y = OF.orthogonalize(x)
    wide = x if shape[0] < shape[1] else x.t()
    m, n = wide.shape
    # X is a polynomial of its Gram matrix times itself: columns suffice
    gram = torch.zeros(m, m, dtype=torch.float64, device=dev())
    for part in wide.split(1 << 20, dim=1):
        p = part.double()
        gram += p @ p.t().contiguous()
    norm = gram.trace().sqrt() + 1e-7
    s, u = torch.linalg.eigh(gram.cpu() / norm.cpu() ** 2)
    s = s.clamp_min(0).sqrt()
    a, b, c = OF.NS_QUINTIC
    f = torch.ones_like(s)
    for _ in range(5):
        q = (s * f) ** 2
        f = f * (a + b * q + c * q * q)
    poly = (u * f) @ u.t()
    got = y if shape[0] < shape[1] else y.t()
    for c0 in (0, n // 2, n - 500):
        want = poly @ (wide[:, c0:c0 + 500].double() / norm).cpu()
        assert off(got[:, c0:c0 + 500], want) < NS_TOL


@gpu
def test_two_graphs_of_all_kinds_replay_in_turn():
    """Every way through the kernels, in two captured graphs that live and
    replay beside each other and beside eager calls."""
    mats = [ns_inputs(s, torch.float32, dev()) for s in
            ((64, 576), (40, 4000), (5, 70, 90), (600, 4700), (1300, 4650),
             (2500, 2500), (2050, 8200), (2050, 12000))]
    logits = [lp_inputs(r, c, torch.bfloat16, dev())
              for r, c in ((3, 300007), (700, 1000))]
    norms = [ln_inputs(s, torch.bfloat16, dev())
             for s in ((40, 8192), (3000, 512), (600, 12000))]

    def first():
        out = [OF.orthogonalize(m) for m in mats[::2]]
        for x, lab in logits:
            leaf = x.detach().requires_grad_(True)
            got = OF.label_logprobs(leaf, lab, top=9)
            out += [*got, *torch.autograd.grad(got[:3], leaf, [
                torch.ones_like(t) for t in got[:3]])]
        return [t.detach() for t in out]

    def second():
        out = [OF.orthogonalize(m) for m in mats[1::2]]
        for x, gamma, beta, dy in norms:
            leaves = [t.detach().requires_grad_(True)
                      for t in (x, gamma, beta)]
            y = OF.layernorm(*leaves)
            out += [y, *torch.autograd.grad(y, leaves, dy)]
        return [t.detach() for t in out]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first(), second()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for work in (first, second):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, work()))
    for turn in range(3):
        for t in mats:
            t.mul_(0.5).add_(torch.randn_like(t), alpha=1e-3)
        for x, _ in logits:
            x.copy_(torch.randn_like(x))
        for x, _, _, dy in norms:
            x.copy_(torch.randn_like(x))
            dy.copy_(torch.randn_like(x))
        want = [[t.clone() for t in work()] for work in (first, second)]
        for graph, _ in graphs[::1 - 2 * (turn % 2)]:
            graph.replay()
        torch.cuda.synchronize()
        for (_, held), ref in zip(graphs, want):
            for i, (a, b) in enumerate(zip(held, ref)):
                assert torch.equal(a, b), (turn, i)
