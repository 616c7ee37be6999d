"""Token log probabilities, entropy, top alternatives and their gradient against fp64.

Tolerances: differences to the maximum are exact to 2^-24, the exponentials and the logarithm
to 2^-22, sums of n terms add a few 2^-24, so a log probability may be off by
2^-20 (1 + |lse| + |x_t|) and the entropy by 2^-19 (1 + H).  A gradient is a product with
p = 2^(log2(e) (x - lse)), whose exponent (|x - lse| up to 100 here) is off by at most 2^-17:
2^-16 p (|A| + |gH| (|log p| + H)) + 2^-22 |sparse terms|, plus bf16's unit roundoff, 2^-8, of the result.
"""

import math

import pytest
import torch


def _exact(x, t, top, ignore=-100):
    """fp64 outputs, and the pieces that the tolerances need."""
    x = x.double()
    m = x.amax(-1, keepdim=True)
    empty = m[:, 0] == -math.inf
    ex = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
    lse = torch.where(empty, -math.inf, m[:, 0] + torch.log(ex.sum(-1)))
    z = torch.where(empty[:, None], -math.inf, x - torch.where(empty, 0.0, lse)[:, None])
    lp = z.gather(1, t.clamp(0, x.shape[1] - 1)[:, None])[:, 0]
    lp = torch.where((t < 0) | (t >= x.shape[1]), math.nan, lp)
    lp = torch.where(t == ignore, 0.0, lp)
    p = torch.exp(z)
    plogp = torch.where(p > 0, p * z, 0.0)
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top]
    return lp, -plogp.sum(-1), z.gather(1, order), order, lse, z, p


def _grad(x, t, top, gl, gh, gt, ignore=-100):
    lp, ent, tl, order, lse, z, p = _exact(x, t, top, ignore)
    empty = lse == -math.inf
    given = (t != ignore) & (t >= 0) & (t < x.shape[1]) & ~empty
    gl = torch.where(given, gl.double(), 0.0)
    gh = torch.where(empty, 0.0, gh.double())
    gt = torch.where(empty[:, None], 0.0, gt.double())
    sparse = torch.zeros_like(p).scatter_add_(1, t.clamp(0, x.shape[1] - 1)[:, None], gl[:, None])
    sparse.scatter_add_(1, order, gt)
    zz = torch.where(z == -math.inf, 0.0, z)
    A = gl + gt.sum(-1)
    g = sparse - p * A[:, None] - gh[:, None] * p * (zz + ent[:, None])
    size = p * (A.abs()[:, None] + gh.abs()[:, None] * (zz.abs() + ent[:, None]))
    return g, size, sparse


def _logits(rows, vocab, kind, dtype, device, seed=0):
    g = torch.Generator(device=device).manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g, device=device) * 3
    t = torch.randint(0, vocab, (rows,), generator=g, device=device)
    if kind == "masked":  # few allowed tokens
        keep = torch.rand(rows, vocab, generator=g, device=device) < 0.02
        keep.scatter_(1, t[:, None], True)
        x = torch.where(keep, x, -math.inf)
    elif kind == "lowest":  # a mask of the type's lowest value
        x = torch.where(torch.rand(rows, vocab, generator=g, device=device) < 0.5, torch.finfo(dtype).min, x)
    elif kind == "flat":
        x = torch.full_like(x, 1.5)
    elif kind == "ties":
        x = torch.randint(-2, 3, x.shape, generator=g, device=device).float()
    elif kind == "columns":  # the large logits lie in few columns a stride apart
        far = torch.arange(vocab, device=device) % 8192 < 8
        x = torch.where(far, 20 + torch.rand(rows, vocab, generator=g, device=device), x)
    elif kind == "peak":
        x.scatter_(1, t[:, None], 100.0)
    elif kind == "large":
        x = x * 1000
    return x.to(dtype), t


def _check(x, t, top, device_out, grads=True):
    lp, ent, tl, tt = device_out
    wl, we, wtl, order, lse, z, p = _exact(x, t, top)
    assert lp.dtype == ent.dtype == tl.dtype == torch.float32 and tt.dtype == torch.int64
    assert torch.equal(tt, order)

    def near(got, want, tol):
        fine = torch.isfinite(want)
        assert torch.equal(got[~fine].double().nan_to_num(7.0), want[~fine].nan_to_num(7.0))
        off = (got.double() - want).abs()[fine]
        assert bool((off <= tol.expand_as(want)[fine]).all()), (off / tol.expand_as(want)[fine]).max()

    s = 1 + torch.where(torch.isfinite(lse), lse, 0.0).abs()
    near(lp, wl, 2.0 ** -20 * (s + wl.abs().nan_to_num(0.0, posinf=0.0)))
    near(ent, we, 2.0 ** -19 * (1 + we))
    near(tl, wtl, 2.0 ** -20 * (s[:, None] + wtl.abs().nan_to_num(posinf=0.0)))


def _check_grad(x, t, top, device):
    from myk_llm_b200 import ops

    g = torch.Generator(device=device).manual_seed(9)
    rows = x.shape[0]
    gl, gh = (torch.randn(rows, generator=g, device=device) for _ in range(2))
    gt = torch.randn(rows, top, generator=g, device=device)
    leaf = x.detach().requires_grad_()
    r = ops.token_logprobs(leaf, t, top=top)
    outs, gs = [r.logprobs, r.entropy], [gl, gh]
    if top:
        outs, gs = outs + [r.top_logprobs], gs + [gt]
    got, = torch.autograd.grad(outs, leaf, gs)
    want, size, sparse = _grad(x, t, top, gl, gh, gt)
    tol = 2.0 ** -16 * size + 2.0 ** -22 * sparse.abs() + 2.0 ** -126
    if x.dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * (want.abs() + tol)
    assert got.dtype == x.dtype and got.shape == x.shape
    off = (got.double() - want).abs()
    assert bool((off <= tol).all()), (off / tol).max()


CASES = [
    # (rows, vocab, top, kind)
    (3, 1, 1, "normal"),
    (2, 5, 5, "normal"),
    (4, 33, 32, "ties"),
    (5, 257, 20, "normal"),
    (3, 1000, 7, "masked"),
    (2, 4096, 32, "flat"),
    (2, 50001, 32, "flat"),
    (2, 65536, 20, "masked"),
    (3, 16383, 10, "ties"),
    (2, 131072, 32, "columns"),
    (2, 400000, 5, "normal"),
    (7, 32768, 0, "normal"),
    (3, 8191, 3, "peak"),
    (3, 777, 4, "lowest"),
    (2, 3001, 4, "large"),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("case", [c for c in CASES if c[1] < 70000])
def test_logprobs_cpu(case, dtype):
    from myk_llm_b200 import ops

    rows, vocab, top, kind = case
    x, t = _logits(rows, vocab, kind, dtype, "cpu")
    _check(x, t, top, ops.token_logprobs(x, t, top=top))
    _check_grad(x, t, top, "cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("case", CASES)
def test_logprobs_gpu(case, dtype):
    from myk_llm_b200 import ops

    rows, vocab, top, kind = case
    x, t = _logits(rows, vocab, kind, dtype, "cuda")
    _check(x, t, top, ops.token_logprobs(x, t, top=top))
    _check_grad(x, t, top, "cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 2, 17, 64, 600])
def test_row_counts(rows):
    """From one row (split over CTAs or not) to many."""
    from myk_llm_b200 import ops

    x, t = _logits(rows, 20011, "normal", torch.bfloat16, "cuda", seed=rows)
    _check(x, t, 20, ops.token_logprobs(x, t, top=20))
    _check(x, t, 0, ops.token_logprobs(x, t))
    _check_grad(x, t, 20, "cuda")


def _special(device):
    from myk_llm_b200 import ops

    v = 5000
    x, t = _logits(8, v, "normal", torch.float32, device)
    x[0] = -math.inf                       # no distribution
    x[1, 1:] = -math.inf                   # one possible token
    t[1] = 0
    x[2, t[2]] = -math.inf                 # the given token is excluded
    t[3] = -100                            # ignored
    t[4] = v                               # outside the vocabulary
    t[5] = -3
    x[6, :100] = -0.0                      # equal to 0
    x[6, 100:] = -1.0
    x[6, 50] = 0.0
    x[7, 2500] = math.nan
    r = ops.token_logprobs(x, t, top=4)
    fine = torch.arange(7, device=device)
    wl, we, wtl, order, *_ = _exact(x[fine], t[fine], 4)
    assert torch.equal(r.top_tokens[fine], order)
    assert r.logprobs[0] == -math.inf and r.entropy[0] == 0 and (r.top_logprobs[0] == -math.inf).all()
    assert r.logprobs[1] == 0 and r.entropy[1] == 0 and (r.top_logprobs[1, 1:] == -math.inf).all()
    assert r.logprobs[2] == -math.inf and r.logprobs[3] == 0
    assert r.logprobs[4].isnan() and r.logprobs[5].isnan() and not r.entropy[4:6].isnan().any()
    assert torch.equal(r.top_tokens[6].cpu(), torch.arange(4))
    assert r.logprobs[7].isnan() and r.entropy[7].isnan() and r.top_logprobs[7].isnan().all()
    # gradients: none for the empty row, the ignored and the impossible tokens
    leaf = x.clone().requires_grad_()
    r = ops.token_logprobs(leaf, t, top=4)
    g, = torch.autograd.grad(r.logprobs[:6].nan_to_num(0.0, neginf=0.0).sum(), leaf)
    assert not g[0].any() and not g[3].any() and not g[4].any() and not g[5].any() and not g[:6].isnan().any()


def test_special_rows_cpu():
    _special("cpu")


@pytest.mark.gpu
def test_special_rows_gpu():
    _special("cuda")


def _infinite(device, dtype, vocab, lo):
    """+inf wherever it lies in a row (first, in the middle, last; alone or beside -inf and NaN) makes the row's
    numbers and gradient NaN and touches no other row; -inf throughout stays "no distribution"."""
    from myk_llm_b200 import ops

    top = min(3, vocab)
    at = sorted({0, 1 % vocab, 7 % vocab, vocab // 2, vocab - 9 if vocab > 9 else 0, vocab - 2 if vocab > 1 else 0, vocab - 1})
    rows = 2 * len(at) + 3
    wide = torch.zeros(rows, vocab + lo + 5, dtype=dtype, device=device)
    x = wide[:, lo:lo + vocab]
    data, t = _logits(rows, vocab, "normal", dtype, device, seed=7)
    x.copy_(data)
    for i, j in enumerate(at):
        x[i, j] = math.inf
        x[len(at) + i] = -math.inf
        x[len(at) + i, j] = math.inf
    x[-1] = -math.inf
    x[-2] = -math.inf
    x[-2, vocab - 1] = math.nan
    bad = torch.arange(rows, device=device) < 2 * len(at)
    bad[-2] = True
    sound = torch.tensor([rows - 3], device=device)
    leaf = x.detach().requires_grad_()
    r = ops.token_logprobs(leaf, t, top=top)
    for y in r[:3]:
        assert y[bad].isnan().all() and not y[~bad].isnan().any()
    for i, j in enumerate(at):
        assert r.top_tokens[i, 0] == j and r.top_tokens[len(at) + i, 0] == j
    _check(x[sound], t[sound], top, [y.detach()[sound] for y in r])
    assert r.logprobs[-1] == -math.inf and r.entropy[-1] == 0 and (r.top_logprobs[-1] == -math.inf).all()
    for out in (r.logprobs, r.entropy, r.top_logprobs):
        g, = torch.autograd.grad(out[:-1].sum(), leaf, retain_graph=True)
        assert g[bad].isnan().all() and not g[~bad].isnan().any() and not g[-1].any()


INFINITE = [(1, 0), (2, 1), (9, 0), (37, 3), (1000, 1), (4099, 0), (20011, 5)]  # (vocabulary, offset of the rows)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab,lo", INFINITE)
def test_infinite_logits_cpu(vocab, lo, dtype):
    _infinite("cpu", dtype, vocab, lo)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab,lo", INFINITE)
def test_infinite_logits_gpu(vocab, lo, dtype):
    _infinite("cuda", dtype, vocab, lo)


def _shifted(device, vocab, shift):
    """Logits far from 0.  They are multiples of 2^-3 below 2^20, so differences to the maximum are exact in fp32 and a
    shift changes no result: a log probability (x_t - m) - log S may be off by 2^-20 (1 + |logprob|), the entropy by
    2^-19 (1 + H), whatever the size of the logits, and the gradient as everywhere in this file."""
    from myk_llm_b200 import ops

    rows, top = 5, min(6, vocab)
    g = torch.Generator(device=device).manual_seed(3)
    x = torch.randint(-80, 81, (rows, vocab), generator=g, device=device) * 0.125 + shift
    t = torch.randint(0, vocab, (rows,), generator=g, device=device)
    r = ops.token_logprobs(x, t, top=top)
    wl, we, wtl, order, *_ = _exact(x - shift, t, top)
    assert torch.equal(r.top_tokens, order)
    for got, want, tol in ((r.logprobs, wl, 2.0 ** -20), (r.entropy, we, 2.0 ** -19), (r.top_logprobs, wtl, 2.0 ** -20)):
        assert bool(((got.double() - want).abs() <= tol * (1 + want.abs())).all())
    _check_grad(x, t, top, device)


SHIFTED = [(v, s) for v in (3, 1000, 40001) for s in (0.0, 2.0 ** 17, -(2.0 ** 19))]


@pytest.mark.parametrize("vocab,shift", SHIFTED)
def test_shifted_logits_cpu(vocab, shift):
    _shifted("cpu", vocab, shift)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab,shift", SHIFTED)
def test_shifted_logits_gpu(vocab, shift):
    _shifted("cuda", vocab, shift)


def _differences(device):
    """The gradient along random directions against central differences in fp64."""
    from myk_llm_b200 import ops

    rows, vocab, top = 6, 301, 5
    x, t = _logits(rows, vocab, "normal", torch.float32, device, seed=4)
    g = torch.Generator(device=device).manual_seed(1)
    gl, gh = (torch.randn(rows, generator=g, device=device) for _ in range(2))
    gt = torch.randn(rows, top, generator=g, device=device)

    def value(y):
        lp, ent, tl, *_ = _exact(y, t, top)
        return (lp * gl).sum() + (ent * gh).sum() + (tl * gt).sum()

    leaf = x.clone().requires_grad_()
    r = ops.token_logprobs(leaf, t, top=top)
    got, = torch.autograd.grad([r.logprobs, r.entropy, r.top_logprobs], leaf, [gl, gh, gt])
    for _ in range(5):
        d = torch.randn(rows, vocab, generator=g, device=device).double()
        h = 1e-5  # truncation h^2 ~ 1e-10, cancellation 1e-16 / h ~ 1e-11
        want = (value(x.double() + h * d) - value(x.double() - h * d)) / (2 * h)
        have = (got.double() * d).sum()
        assert abs(have - want) <= 1e-5 * (got.double() * d).abs().sum() + 1e-8


def test_gradient_differences_cpu():
    _differences("cpu")


@pytest.mark.gpu
def test_gradient_differences_gpu():
    _differences("cuda")


def _in_place(device):
    """Outputs masked in place before backward: the gradient of the masked values."""
    from myk_llm_b200 import ops

    x, t = _logits(12, 503, "normal", torch.float32, device)
    pad = torch.arange(12, device=device) % 3 == 0
    for shape in ((12,), (3, 4)):
        grads = []
        for in_place in (False, True):
            leaf = x.clone().requires_grad_()
            r = ops.token_logprobs(leaf.view(*shape, 503), t.view(shape), top=4)
            lp, ent, tl = r.logprobs, r.entropy, r.top_logprobs
            mask = pad.view(shape)
            if in_place:
                lp.masked_fill_(mask, 0.0)
                lp.mul_(2.0)
                ent[mask] = 0.0
                tl.clamp_(min=-4.0)
            else:
                lp = 2.0 * lp.masked_fill(mask, 0.0)
                ent = ent.masked_fill(mask, 0.0)
                tl = tl.clamp(min=-4.0)
            grads.append(torch.autograd.grad(lp.sum() + 0.1 * ent.sum() + tl.sum(), leaf)[0])
        assert torch.equal(*grads)


def test_outputs_in_place_cpu():
    _in_place("cpu")


@pytest.mark.gpu
def test_outputs_in_place_gpu():
    _in_place("cuda")


@pytest.mark.gpu
def test_second_derivative_is_refused():
    """The kernels have a first derivative; differentiating it again is an error, not a wrong gradient."""
    from myk_llm_b200 import ops

    x, t = _logits(5, 101, "normal", torch.float32, "cuda")
    leaf = x.clone().requires_grad_()
    g, = torch.autograd.grad(ops.token_logprobs(leaf, t).logprobs.sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        (g.square().sum() + 0.0 * leaf.sum()).backward()


@pytest.mark.gpu
def test_shapes_strides_and_partial_gradients():
    """Batched shapes, padded vocabularies (rows apart, unaligned), transposed logits, int32
    tokens, another stream, and gradients through one output alone."""
    from myk_llm_b200 import ops

    x, t = _logits(12, 1003, "normal", torch.bfloat16, "cuda")
    base = ops.token_logprobs(x, t, top=6)
    r = ops.token_logprobs(x.view(3, 4, 1003), t.view(3, 4).int(), top=6)
    assert all(torch.equal(a.reshape(b.shape), b) for a, b in zip(r, base))
    assert r.top_tokens.shape == (3, 4, 6)
    for pad, lo in ((5, 0), (5, 3), (1021, 8)):
        wide = torch.randn(12, 1003 + pad + lo, device="cuda").to(torch.bfloat16) + 50
        view = wide[:, lo:lo + 1003]
        view.copy_(x)
        r = ops.token_logprobs(view, t, top=6)
        _check(x, t, 6, r)
        _check_grad(view, t, 6, "cuda")
    r = ops.token_logprobs(x.t().contiguous().t(), t, top=6)
    assert all(torch.equal(a, b) for a, b in zip(r, base))
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        r = ops.token_logprobs(x, t, top=6)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(r, base))
    leaf = x.clone().requires_grad_()
    one = torch.ones(12, device="cuda")
    for name, gl, gh in (("logprobs", one, 0 * one), ("entropy", 0 * one, one)):
        got, = torch.autograd.grad(getattr(ops.token_logprobs(leaf, t, top=6), name).sum(), leaf)
        want, size, _ = _grad(x, t, 6, gl, gh, torch.zeros(12, 6, device="cuda"))
        assert bool(((got.double() - want).abs() <= 2.0 ** -8 * (want.abs() + 2.0 ** -16 * size) + 2.0 ** -16 * size).all())
    assert not ops.token_logprobs(leaf, t).top_tokens.requires_grad
    empty = ops.token_logprobs(x[:0], t[:0], top=3)
    assert empty.logprobs.shape == (0,) and empty.top_tokens.shape == (0, 3)


def test_refusals():
    from myk_llm_b200 import ops

    x, t = torch.zeros(3, 10), torch.zeros(3, dtype=torch.long)
    for bad in (dict(top=11), dict(top=-1)):
        with pytest.raises(ValueError):
            ops.token_logprobs(x, t, **bad)
    with pytest.raises(ValueError):
        ops.token_logprobs(torch.zeros(3, 100), t, top=33)
    with pytest.raises(ValueError):
        ops.token_logprobs(x, t[:2])
    with pytest.raises(TypeError):
        ops.token_logprobs(x, t.float())


@pytest.mark.gpu
def test_kernel_refusals():
    from myk_llm_b200 import ops

    x, t = torch.zeros(3, 10, device="cuda"), torch.zeros(3, dtype=torch.long, device="cuda")
    with pytest.raises(TypeError):
        ops.token_logprobs(x.half(), t)
    with pytest.raises(RuntimeError):
        ops.token_logprobs(x, t.cpu())
