"""Token-model operators against plain implementations in 64 bits. Tolerances count roundings: u = 2^-24 for an fp32
operation, finfo.eps / 2 for the rounding to the stored type, and the length of the longest chain of additions."""
import ctypes
import math
import os

import pytest
import torch

import neuzephyr_b200 as nz
from neuzephyr_b200 import _capi as C

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]


def rnd(shape, seed, dtype=F32, std=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=g) * std).to(dtype)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def within(got, want, tol):
    """|got - want| <= tol, element by element; equal where not finite."""
    got, want = got.double(), want.double()
    tol = torch.as_tensor(tol, dtype=torch.float64, device=got.device).expand_as(want)
    assert got.shape == want.shape
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)])
    bad = ((got - want).abs() > tol) & fine
    assert not bad.any(), "worst excess %g at %s" % ((((got - want).abs() / tol)[fine]).max(), bad.nonzero()[0].tolist())


def padded(t, extra, offset=0):
    """The matrix t with `extra` more elements between its rows, starting `offset` elements into its memory."""
    rows, cols = t.shape
    buf = torch.full((offset + rows * (cols + extra),), 77.0, dtype=F32, device=t.device).to(t.dtype)
    v = buf[offset:].view(rows, cols + extra)[:, :cols]
    v.copy_(t)
    return v


# ---- embedding ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("tokens,vocab,dim", [(1, 1, 1), (1, 7, 8), (3, 100, 64), (17, 50, 130), (33, 1000, 883), (257, 300, 2048),
                                              (5, 4, 4099)])
@pytest.mark.parametrize("dtype", TYPES)
def test_embedding(tokens, vocab, dim, dtype):
    table = rnd((vocab, dim), 1, dtype)
    idx = torch.randint(0, vocab, (tokens,), device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    idx[0] = vocab - 1
    for index in (idx, idx.int()):
        for scale in (1.0, 1.7):
            want = table[idx].double() * scale
            # one product in fp32 and one rounding to the type; scale itself is rounded to fp32
            tol = want.abs() * (half_step(dtype) + 2.1 * U) + 2.0 ** -25
            within(nz.embedding(table, index, scale=scale), want, tol)
    if dtype != F32:
        wide = rnd((vocab, dim), 3)
        want = wide[idx].double() * 0.37
        within(nz.embedding(wide, idx, scale=0.37, out_dtype=dtype), want, want.abs() * (half_step(dtype) + 2.1 * U) + 2.0 ** -25)


def test_embedding_outside_strides_and_shapes():
    table = rnd((40, 24), 4)
    idx = torch.tensor([[0, -1, 39], [40, 7, 2 ** 40]], device="cuda")
    got = nz.embedding(table, idx, scale=2.0)
    want = torch.zeros(2, 3, 24, device="cuda")
    for i, j in ((0, 0), (0, 2), (1, 1)):
        want[i, j] = table[idx[i, j]] * 2.0
    assert torch.equal(got, want)
    for extra, offset in ((3, 0), (4, 0), (4, 1), (8, 4)):
        view, out = padded(table, extra, offset), padded(torch.zeros(5, 24, device="cuda"), extra, offset)
        i5 = torch.tensor([3, 3, 0, 39, 11], device="cuda", dtype=torch.int32)
        before = out._base.clone()
        nz.embedding(view, i5, out=out)
        assert torch.equal(out, table[i5.long()])
        out.copy_(padded(torch.zeros(5, 24, device="cuda"), 0))
        assert torch.equal(out._base, before)  # nothing between the rows was written
    assert nz.embedding(table, torch.empty(0, dtype=torch.int64, device="cuda")).shape == (0, 24)


def _embedding_grad(dy, idx, vocab, scale, padding):
    """The sums in 64 bits, the sums of magnitudes and the number of addends."""
    keep = (idx >= 0) & (idx < vocab)
    if padding is not None:
        keep &= idx != padding
    at = idx[keep].long()
    d = dy.double()[keep] * scale
    zero = torch.zeros(vocab, dy.shape[1], dtype=torch.float64, device="cuda")
    return zero.index_add(0, at, d), zero.index_add(0, at, d.abs()), torch.bincount(at, minlength=vocab)[:, None]


@pytest.mark.parametrize("tokens,vocab,dim", [(1, 1, 1), (1, 300, 64), (64, 3, 40), (65, 3, 40), (200, 2, 257), (1000, 70000, 24),
                                              (2048, 300, 16), (2049, 300, 16), (3000, 5000, 200), (16384, 500, 16), (16385, 500, 16),
                                              (40000, 33, 12), (5000, 1 << 20, 8)])
@pytest.mark.parametrize("dtype", TYPES)
def test_embedding_backward(tokens, vocab, dim, dtype):
    g = torch.Generator("cuda").manual_seed(5)
    idx = (torch.rand(tokens, device="cuda", generator=g) ** 3 * vocab).long().clamp_(max=vocab - 1)
    if tokens > 3:
        idx[1], idx[2] = -100, vocab
    dy = rnd((tokens, dim), 6, dtype)
    padding = int(idx[0]) if tokens > 100 else None
    want, mags, count = _embedding_grad(dy, idx, vocab, 1.3, padding)
    tol = mags * (count + 6) * U + 1e-30  # count - 1 additions, the scale's rounding and product, joins of pieces
    out = torch.full((vocab, dim), float("nan"), device="cuda")
    nz.embedding_backward(dy, idx, out, scale=1.3, padding_index=padding, overwrite=True)
    within(out, want, tol)
    again = torch.full((vocab, dim), 7.0, device="cuda")
    nz.embedding_backward(dy, idx.int(), again, scale=1.3, padding_index=padding, overwrite=True)
    assert torch.equal(out, again)  # the same bits, whatever the buffer held and the index type
    start = rnd((vocab, dim), 7)
    added = start.clone()
    nz.embedding_backward(dy, idx, added, scale=1.3, padding_index=padding)
    within(added, start.double() + want, tol + (start.abs() + mags) * (2 + tokens // 16384) * U)
    untouched = count[:, 0] == 0
    assert torch.equal(added[untouched], start[untouched])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_embedding_backward_strides_and_empty(dtype):
    vocab, dim, tokens = 50, 40, 300
    idx = torch.randint(0, vocab, (tokens,), device="cuda", generator=torch.Generator("cuda").manual_seed(8))
    dy = rnd((tokens, dim), 9, dtype)
    plain = torch.empty(vocab, dim, device="cuda")
    nz.embedding_backward(dy, idx, plain, overwrite=True)
    for extra, offset in ((3, 0), (8, 0), (8, 1), (16, 8)):
        out = padded(torch.zeros(vocab, dim, device="cuda"), extra, offset)
        before = out._base.clone()
        nz.embedding_backward(padded(dy, extra, offset), idx, out, overwrite=True)
        assert torch.equal(out, plain)
        out.zero_()
        assert torch.equal(out._base, before)
    nz.embedding_backward(dy[:0], idx[:0], plain, overwrite=True)
    assert torch.equal(plain, torch.zeros_like(plain))
    all_padding = torch.full((tokens,), 3, device="cuda")
    plain.fill_(float("nan"))
    nz.embedding_backward(dy, all_padding, plain, padding_index=3, overwrite=True)
    assert torch.equal(plain, torch.zeros_like(plain))
    # a linear function: its differences are the gradient itself
    table = rnd((vocab, dim), 10)
    moved = table.clone()
    moved[idx[5], 3] += 0.5
    w = dy.float()
    rise = ((nz.embedding(moved, idx).double() - nz.embedding(table, idx).double()) * w.double()).sum() / 0.5
    nz.embedding_backward(w, idx, plain, overwrite=True)
    within(plain[idx[5], 3], rise, 1e-4)  # table entries near 1 rounded to 2^-24, over a step of 0.5, times |w| sums of about 30


# ---- layer norm --------------------------------------------------------------------------------------------
CHAIN = 96  # additions a sum over a row goes through at most: 32 in a thread, 5 shuffles, 32 warps, centring


def _norm_ref(x, gamma, beta, eps):
    x = x.double()
    mean = x.mean(1, keepdim=True)
    var = (x - mean).square().mean(1, keepdim=True)
    rstd = (var + eps).rsqrt()
    h = (x - mean) * rstd
    g = 1.0 if gamma is None else gamma.double()
    return h * g + (0.0 if beta is None else beta.double()), mean, rstd, h, g


def _check_norm(x, gamma, beta, eps, got):
    y, mean, rstd, h, g = _norm_ref(x, gamma, beta, eps)
    mean_tol = CHAIN * U * x.double().abs().mean(1, keepdim=True) + 1e-37
    # an error of the mean enters the variance squared only, beside the roundings of the centred values
    rstd_tol = rstd * (CHAIN * U + 2 * (mean_tol * rstd) ** 2) + 1e-37
    within(got[1], mean[:, 0], mean_tol[:, 0])
    within(got[2], rstd[:, 0], rstd_tol[:, 0])
    g = torch.as_tensor(g, device="cuda").abs()
    tol = g * rstd * (mean_tol + 2 * U * x.double().abs()) + (g * h.abs()) * (rstd_tol / rstd + 4 * U) + 2 * U * y.abs()
    if beta is not None:
        tol = tol + U * beta.double().abs()
    within(got[0], y, tol + half_step(got[0].dtype) * (y.abs() + tol) + 2.0 ** -25)


@pytest.mark.parametrize("rows,dim", [(1, 1), (1, 2), (3, 7), (2, 64), (5, 100), (4, 129), (9, 257), (64, 1024), (7, 1025), (3, 2050),
                                      (5, 4096), (3, 5003), (2, 8192), (2, 16000), (1, 32768), (2, 40001)])
@pytest.mark.parametrize("dtype", TYPES)
def test_layernorm_forward(rows, dim, dtype):
    x = (rnd((rows, dim), 11) * 2 + rnd((rows, 1), 12) * 5).to(dtype)
    gamma, beta = rnd((dim,), 13) + 1, rnd((dim,), 14)
    _check_norm(x, gamma, beta, 1e-5, nz.layernorm_forward(x, gamma, beta))
    _check_norm(x, None, None, 1e-3, nz.layernorm_forward(x, eps=1e-3))
    for extra, offset in ((1, 0), (8, 1), (8, 8)):
        xv = padded(x, extra, offset)
        _check_norm(x, gamma, None, 1e-5, nz.layernorm_forward(xv, gamma))
        out = padded(torch.zeros_like(x), 8, 0)
        before = out._base.clone()
        _check_norm(x, gamma, beta, 1e-5, nz.layernorm_forward(xv, gamma, beta, out=out))
        out.zero_()
        assert torch.equal(out._base, before)
    inplace = x.clone()
    want = nz.layernorm_forward(x, gamma, beta)[0]
    assert torch.equal(nz.layernorm_forward(inplace, gamma, beta, out=inplace)[0], want) and torch.equal(inplace, want)


def test_layernorm_special_rows():
    x = rnd((6, 300), 15)
    x[0] = 3.0          # no spread: y = beta
    x[1] = 1e4 + x[1]   # a large mean
    x[2] = 0.0
    x[3, 7] = float("nan")
    x[4, 9] = float("inf")
    y, mean, rstd = nz.layernorm_forward(x)
    assert torch.equal(y[0], torch.zeros(300, device="cuda")) and mean[0] == 3.0
    assert torch.equal(y[2], torch.zeros(300, device="cuda"))
    assert torch.isnan(y[3]).all() and torch.isnan(y[4]).any()
    keep = torch.tensor([0, 1, 2, 5], device="cuda")
    _check_norm(x[keep], None, None, 1e-5, (y[keep], mean[keep], rstd[keep]))
    assert nz.layernorm_forward(x[:0])[0].shape == (0, 300)


def _norm_grads(dy, x, mean, rstd, gamma):
    h = (x.double() - mean.double()[:, None]) * rstd.double()[:, None]
    d = dy.double()
    g = d * (1.0 if gamma is None else gamma.double())
    r = rstd.double()[:, None]
    dx = r * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
    hm = h.abs() + 2 * r * (x.double().abs() + mean.double().abs()[:, None])  # what the roundings of x - mean scale with
    mags = r * (g.abs() + g.abs().mean(1, keepdim=True) + hm * (g.abs() * hm).mean(1, keepdim=True))
    return dx, mags * 2 * CHAIN * U, (d * h).sum(0), (d.abs() * hm).sum(0), d.sum(0), d.abs().sum(0)


@pytest.mark.parametrize("rows,dim", [(1, 1), (1, 5), (3, 64), (50, 96), (7, 129), (300, 257), (64, 1024), (33, 2050), (700, 100),
                                      (40, 4096), (21, 5003), (3, 8192), (17, 16000), (2, 20001)])
@pytest.mark.parametrize("dtype", TYPES)
def test_layernorm_backward(rows, dim, dtype):
    x = (rnd((rows, dim), 16) * 2 + rnd((rows, 1), 17)).to(dtype)
    dy, gamma = rnd((rows, dim), 18, dtype), rnd((dim,), 19) + 1
    _, mean, rstd = nz.layernorm_forward(x, gamma)
    for gm in (gamma, None):
        dx, dx_tol, dg, dg_mags, db, db_mags = _norm_grads(dy, x, mean, rstd, gm)
        chain = rows + 32
        outs = torch.full_like(x, float("nan")), torch.full((dim,), float("nan"), device="cuda"), torch.full((dim,), float("nan"), device="cuda")
        nz.layernorm_backward(dy, x, mean, rstd, gm, *outs, overwrite_dx=True, overwrite_dparams=True)
        within(outs[0], dx, dx_tol + half_step(dtype) * (dx.abs() + dx_tol) + 2.0 ** -25)
        within(outs[1], dg, dg_mags * chain * U + 1e-30)
        within(outs[2], db, db_mags * chain * U + 1e-30)
        # added to what is there
        base = rnd((rows, dim), 20, dtype), rnd((dim,), 21), rnd((dim,), 22)
        acc = [t.clone() for t in base]
        nz.layernorm_backward(dy, x, mean, rstd, gm, *acc)
        total = base[0].double() + dx
        within(acc[0], total, dx_tol + 2 * U * (total.abs() + dx.abs()) + half_step(dtype) * (total.abs() + dx_tol) + 2.0 ** -25)
        within(acc[1], base[1].double() + dg, (dg_mags + base[1].abs()) * (chain + 2) * U + 1e-30)
        within(acc[2], base[2].double() + db, (db_mags + base[2].abs()) * (chain + 2) * U + 1e-30)
        # the same bits with any part left out, with other strides, and in place
        only = torch.empty(dim, device="cuda")
        nz.layernorm_backward(dy, x, mean, rstd, gm, dgamma=only, overwrite_dparams=True)
        within(only, dg, dg_mags * chain * U + 1e-30)
        nz.layernorm_backward(dy, x, mean, rstd, gm, dbeta=only, overwrite_dparams=True)
        within(only, db, db_mags * chain * U + 1e-30)
        for extra, offset, other in ((1, 0, 1), (8, 8, 8), (8, 1, 3)):
            dxv = padded(torch.zeros_like(x), other, offset)
            before = dxv._base.clone()
            nz.layernorm_backward(padded(dy, extra, offset), padded(x, extra, offset), mean, rstd, gm, dxv, outs[1], outs[2],
                                  overwrite_dx=True, overwrite_dparams=True)
            within(dxv, dx, dx_tol + half_step(dtype) * (dx.abs() + dx_tol) + 2.0 ** -25)
            within(outs[1], dg, dg_mags * chain * U + 1e-30)
            dxv.zero_()
            assert torch.equal(dxv._base, before)
        inplace = dy.clone()
        nz.layernorm_backward(inplace, x, mean, rstd, gm, inplace, overwrite_dx=True)
        assert torch.equal(inplace, outs[0])


def test_layernorm_backward_of_no_rows():
    x = torch.empty(0, 12, device="cuda")
    v = torch.ones(12, device="cuda")
    nz.layernorm_backward(x, x, v[:0], v[:0], None, None, v, None, overwrite_dparams=True)
    assert torch.equal(v, torch.zeros(12, device="cuda"))
    v.fill_(1)
    nz.layernorm_backward(x, x, v[:0], v[:0], None, None, v, None)
    assert torch.equal(v, torch.ones(12, device="cuda"))


def test_layernorm_gradient_against_differences():
    rows, dim, step = 3, 40, 2.0 ** -6
    x, gamma, beta, w = rnd((rows, dim), 23), rnd((dim,), 24) + 1, rnd((dim,), 25), rnd((rows, dim), 26)
    _, mean, rstd = nz.layernorm_forward(x, gamma, beta)
    dx, dg, db = torch.empty_like(x), torch.empty(dim, device="cuda"), torch.empty(dim, device="cuda")
    nz.layernorm_backward(w, x, mean, rstd, gamma, dx, dg, db, overwrite_dx=True, overwrite_dparams=True)

    def loss(x, gamma, beta):
        return (nz.layernorm_forward(x, gamma, beta)[0].double() * w.double()).sum()
    # central differences: rounding noise of 120 values near 1 over 2 steps, 120 * 16 u * |w| / 2^-5 < 0.01, and a third
    # derivative of order 10 times step^2 / 6 < 1e-3
    for r, c in ((0, 0), (1, 17), (2, 39)):
        e = torch.zeros_like(x)
        e[r, c] = step
        within((loss(x + e, gamma, beta) - loss(x - e, gamma, beta)) / (2 * step), dx[r, c].double(), 0.011)
        e = torch.zeros_like(gamma)
        e[c] = step
        within((loss(x, gamma + e, beta) - loss(x, gamma - e, beta)) / (2 * step), dg[c].double(), 0.011)
        within((loss(x, gamma, beta + e) - loss(x, gamma, beta - e)) / (2 * step), db[c].double(), 0.011)


# ---- token log probabilities -------------------------------------------------------------------------------
def _logprob_ref(x, t, scale, k):
    z = x.double() * scale
    lse = torch.logsumexp(z, 1)
    logq = z - lse[:, None]
    p = logq.exp()
    ent = -torch.where(p > 0, p * logq, 0.0).sum(1)
    inside = (t >= 0) & (t < x.shape[1])
    lp = torch.where(inside, logq.gather(1, torch.where(inside, t, 0).long()[:, None])[:, 0], 0.0)
    order = torch.sort(x.double(), dim=1, descending=True, stable=True)[1][:, :k]
    return lp, ent, lse, logq.gather(1, order), order


def _sums_tol(vocab):
    """Relative error of sum exp: the exponential's 2^-22, two roundings of its argument (weighted by at most ln vocab
    + 4), additions of a thread's share and of the joins."""
    return 2.0 ** -22 + 2 * U * (math.log(vocab) + 4) * 2 + (vocab / 256 + 48) * U


def _check_logprob(x, t, scale, k, got):
    lp, ent, lse, top, order = _logprob_ref(x, t, scale, k)
    s = _sums_tol(x.shape[1])
    within(got.lse, lse, s + 4 * U * lse.abs())
    within(got.logprob, lp, s + 8 * U * (lp.abs() + 1))
    within(got.entropy, ent, 2 * s * (2 + ent) + 4 * U * ent)
    within(got.top_logprob, top, s + 8 * U * (top.abs() + 1))
    assert torch.equal(got.top_index.long(), order)


@pytest.mark.parametrize("rows,vocab,k", [(1, 1, 1), (1, 1, 0), (2, 3, 3), (3, 33, 5), (5, 300, 32), (4, 1000, 8), (7, 4099, 20), (2, 50021, 5),
                                          (1, 131072, 32), (300, 777, 4), (3, 200001, 1)])
@pytest.mark.parametrize("dtype", TYPES)
def test_token_logprobs(rows, vocab, k, dtype):
    x = (rnd((rows, vocab), 27) * 3).to(dtype)
    t = torch.randint(0, vocab, (rows,), device="cuda", generator=torch.Generator("cuda").manual_seed(28))
    if rows > 2:
        t[1], t[2] = -100, vocab
    for scale in (1.0, 0.7):
        _check_logprob(x, t, scale, k, nz.token_logprobs(x, t, scale=scale, top_k=k))
    for extra, offset in ((1, 0), (8, 1)):
        got = nz.token_logprobs(padded(x, extra, offset), t.int(), top_k=k)
        _check_logprob(x, t, 1.0, k, got)
        assert got.top_index.dtype == torch.int32


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [40, 1000, 9001])
def test_token_logprobs_masks(dtype, vocab):
    lowest = torch.finfo(dtype).min
    x = rnd((12, vocab), 29, dtype)
    x[0, :] = -math.inf
    x[0, vocab // 2] = 2.0                 # one token left
    x[1, : vocab - 5] = -math.inf          # five left, fewer than the alternatives asked for
    x[2, 3:] = lowest
    x[3, :] = 0.25                         # all equal: alternatives in order of their columns
    x[4, :] = -math.inf                    # nothing left
    x[5, ::2] = -math.inf
    x[6, 1:] = x[6, 0]                     # equal to the first
    x[7, vocab - 1] = 60.0                 # one token takes all
    x[8] = x[8].abs().neg() * 1000 if dtype != F16 else x[8].abs().neg() * 100
    x[9] = torch.arange(vocab, device="cuda").to(dtype)  # rising: the largest are neighbours
    x[10] = torch.arange(vocab, 0, -1, device="cuda").to(dtype)
    t = torch.full((12,), vocab // 2, device="cuda")
    got = nz.token_logprobs(x, t, top_k=8)
    keep = torch.tensor([i for i in range(12) if i != 4], device="cuda")
    pick = lambda g: type(g)(*(v[keep] for v in g))
    lp, ent, lse, top, order = _logprob_ref(x[keep], t[keep], 1.0, 8)
    s = _sums_tol(vocab)
    g = pick(got)
    within(g.lse, lse, s + 4 * U * lse.abs())
    within(g.entropy, ent, 2 * s * (2 + ent) + 4 * U * ent)
    within(g.logprob, lp, s + 8 * U * (lp.abs() + 1))
    within(g.top_logprob, top, s + 8 * U * (top.abs() + 1))
    assert torch.equal(g.top_index, order)
    assert got.lse[4] == -math.inf and got.logprob[4] == -math.inf and got.entropy[4] == 0
    assert (got.top_logprob[4] == -math.inf).all() and torch.equal(got.top_index[4], torch.arange(8, device="cuda"))
    # every logit at the type's lowest value: of fp32 and bf16 below any z that counts, of fp16 an ordinary number
    x[0, :] = lowest
    got = nz.token_logprobs(x, t)
    if dtype == F16:
        within(got.entropy[0], torch.tensor(math.log(vocab), device="cuda"), 2 * s * (2 + math.log(vocab)))
    else:
        assert got.lse[0] == -math.inf and got.entropy[0] == 0 and got.logprob[0] == -math.inf
    # NaN makes its row's numbers NaN and no others; it is no alternative
    x[5, 1] = math.nan
    got = nz.token_logprobs(x, t, top_k=3)
    assert torch.isnan(got.lse[5]) and torch.isnan(got.logprob[5]) and torch.isnan(got.entropy[5])
    assert not torch.isnan(got.lse[6:]).any() and (got.top_index[5] != 1).all()


def _logprob_grad_ref(x, t, lse, ent, dl, dh, scale):
    q = x.double() * scale - lse.double()[:, None]
    p = q.exp()
    inside = ((t >= 0) & (t < x.shape[1]))
    dlv = torch.zeros_like(lse, dtype=torch.float64) if dl is None else torch.where(inside, dl.double(), 0.0)
    dhv = torch.zeros_like(dlv) if dh is None else dh.double()
    H = torch.zeros_like(dlv) if ent is None else ent.double()
    wave = torch.where(p > 0, p * (q + H[:, None]), 0.0)
    d = -dlv[:, None] * p - dhv[:, None] * wave
    d.scatter_add_(1, torch.where(inside, t, 0).long()[:, None], dlv[:, None])
    qa = torch.where(p > 0, q.abs(), 0.0)
    tol = p * (2.0 ** -21 + 2.0 ** -22 * qa) * (dlv.abs()[:, None] + dhv.abs()[:, None] * (qa + H.abs()[:, None]))
    tol.scatter_add_(1, torch.where(inside, t, 0).long()[:, None], 4 * U * dlv.abs()[:, None])
    return d * scale, tol * scale + 2 * U * scale * d.abs() + 2.0 ** -125  # p below fp32's smallest normal number is 0


@pytest.mark.parametrize("rows,vocab", [(1, 1), (2, 3), (3, 33), (5, 1000), (4, 4099), (2, 50021), (1, 131072), (300, 77)])
@pytest.mark.parametrize("dtype", TYPES)
def test_token_logprobs_backward(rows, vocab, dtype):
    x = (rnd((rows, vocab), 30) * 3).to(dtype)
    if vocab > 10:
        x[:, 4:7] = -math.inf
    t = torch.randint(0, vocab, (rows,), device="cuda", generator=torch.Generator("cuda").manual_seed(31))
    if rows > 2:
        t[1], t[2] = -100, 5 if vocab > 10 else vocab  # without a target; with a masked one
    scale = 1.25
    f = nz.token_logprobs(x, t, scale=scale)
    for dl, dh in ((rnd((rows,), 32), None), (None, rnd((rows,), 33)), (rnd((rows,), 32), rnd((rows,), 33))):
        want, tol = _logprob_grad_ref(x, t, f.lse, f.entropy, dl, dh, scale)
        tol = tol + half_step(dtype) * (want.abs() + tol) + (2.0 ** -25 if dtype == F16 else 0.0)
        got = nz.token_logprobs_backward(x, t, f.lse, f.entropy if dh is not None else None, dl, dh, scale=scale)
        within(got, want, tol)
        for extra, offset, other in ((1, 0, 1), (8, 1, 3)):
            out = padded(torch.zeros_like(x), other, offset)
            before = out._base.clone()
            nz.token_logprobs_backward(padded(x, extra, offset), t.int(), f.lse, f.entropy, dl, dh, scale=scale, out=out)
            assert torch.equal(out, got)
            out.zero_()
            assert torch.equal(out._base, before)
        inplace = x.clone()
        nz.token_logprobs_backward(inplace, t, f.lse, f.entropy, dl, dh, scale=scale, out=inplace)
        assert torch.equal(inplace, got)


@pytest.mark.parametrize("dtype", TYPES)
def test_token_logprobs_backward_of_empty_rows(dtype):
    x = rnd((3, 100), 34, dtype)
    x[1] = -math.inf
    t = torch.tensor([5, 6, 7], device="cuda")
    one = torch.ones(3, device="cuda")
    f = nz.token_logprobs(x, t)
    got = nz.token_logprobs_backward(x, t, f.lse, f.entropy, one, one)
    assert torch.equal(got[1], torch.zeros_like(got[1])) and torch.isfinite(got).all()
    assert nz.token_logprobs(x[:0], t[:0], top_k=2).top_index.shape == (0, 2)
    assert nz.token_logprobs_backward(x[:0], t[:0], one[:0], None, one[:0]).shape == (0, 100)


def test_token_logprobs_gradient_against_differences():
    rows, vocab, step = 2, 50, 2.0 ** -5
    x, t = rnd((rows, vocab), 35), torch.tensor([3, 44], device="cuda")
    dl, dh = rnd((rows,), 36), rnd((rows,), 37)
    f = nz.token_logprobs(x, t, scale=1.5)
    d = nz.token_logprobs_backward(x, t, f.lse, f.entropy, dl, dh, scale=1.5)

    def loss(x):
        f = nz.token_logprobs(x, t, scale=1.5)
        return (f.logprob.double() * dl.double() + f.entropy.double() * dh.double()).sum()
    # noise of four values below 8 (2^-20 each) over 2 steps: 4 * 2 * 2^-20 / 2^-4 = 1.3e-4; third derivative of order
    # 1.5^3 * 8 times step^2 / 6: 4.4e-3
    for r, c in ((0, 0), (0, 3), (1, 44), (1, 20)):
        e = torch.zeros_like(x)
        e[r, c] = step
        within((loss(x + e) - loss(x - e)) / (2 * step), d[r, c].double(), 5e-3)


# ---- orthogonalised updates --------------------------------------------------------------------------------
def _ortho_ref(g, steps=5, eps=1e-7):
    a, b, c = nz.ops.NEWTON_SCHULZ
    x = g.double()
    x = x / (torch.linalg.norm(x) + eps)
    tall = x.shape[0] > x.shape[1]
    x = x.mT if tall else x
    for _ in range(steps):
        m = x @ x.mT
        x = a * x + (b * m + c * m @ m) @ x
    return x.mT if tall else x


def _rel(got, want):
    return float(torch.linalg.norm(got.double() - want) / torch.linalg.norm(want))


def _gradient_like(rows, cols, seed):
    n = 2 * max(rows, cols)
    up = rnd((rows, n), seed) * (torch.arange(rows, device="cuda") + 1.0)[:, None] ** -0.5
    act = rnd((n, cols), seed + 1) * (torch.arange(cols, device="cuda") + 1.0) ** -0.5
    return up @ act


# The operands' roundings (2^-12 relative, three products in each of five steps) give at most 2.9e-3 in a simulation in
# 64 bits with only these roundings in it, on full-rank, decaying and nearly low-rank matrices with sides from 64 on;
# twice that, and the rounding of the output, is allowed.
ORTHO_TOL = 6e-3


@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 7), (7, 1), (2, 2), (5, 64), (64, 5), (64, 64), (100, 300), (300, 100), (128, 128), (129, 257),
                                       (257, 129), (256, 512), (1000, 520), (513, 1025), (640, 640), (1030, 1100)])
@pytest.mark.parametrize("dtype", TYPES)
def test_orthogonalize(rows, cols, dtype):
    for g in (_gradient_like(rows, cols, 40).to(dtype), rnd((rows, cols), 42, dtype, std=1e-3)):
        want = _ortho_ref(g)
        for out_dtype in TYPES if dtype == F32 else [dtype]:
            got = nz.orthogonalize(g, out_dtype=out_dtype)
            assert got.dtype == out_dtype and torch.isfinite(got).all()
            assert _rel(got, want) <= ORTHO_TOL + half_step(out_dtype)
        assert torch.equal(got, nz.orthogonalize(g, out_dtype=got.dtype))


@pytest.mark.parametrize("batch,rows,cols", [(1, 130, 5000), (1, 5000, 130), (1, 31, 9001), (1, 700, 4100), (2, 4001, 300), (1, 64, 1030)])
def test_orthogonalize_long_sides(batch, rows, cols):
    """A long contraction of few tiles is shared among CTAs."""
    g = torch.stack([_gradient_like(rows, cols, 47 + i) for i in range(batch)])
    got = nz.orthogonalize(g)
    for i in range(batch):
        assert _rel(got[i], _ortho_ref(g[i])) <= ORTHO_TOL
    assert torch.equal(got, nz.orthogonalize(g))


@pytest.mark.parametrize("rows,cols", [(64, 96), (96, 64), (300, 500), (500, 300)])
def test_orthogonalize_one_step_and_low_rank(rows, cols):
    g = rnd((rows, cols), 43)
    # one step: (B X)'s operands and B's own rounding, |B| <= 2.8 against |X_1| >= 0.7 |X|: 3 * 2^-12 * 4
    assert _rel(nz.orthogonalize(g, steps=1), _ortho_ref(g, steps=1)) <= 3 * 2.0 ** -12 * 4
    low = rnd((rows, 8), 44) @ rnd((8, cols), 45) + 0.01 * g
    assert _rel(nz.orthogonalize(low), _ortho_ref(low)) <= ORTHO_TOL
    one = torch.zeros(rows, cols, device="cuda")
    one[3, 5] = -7.0
    assert _rel(nz.orthogonalize(one), _ortho_ref(one)) <= ORTHO_TOL
    sv = torch.linalg.svdvals(nz.orthogonalize(_gradient_like(rows, cols, 46)).double())
    assert sv.max() < 1.3


def test_orthogonalize_batches_strides_and_extremes():
    for rows, cols in ((100, 140), (140, 100)):
        g = torch.stack([_gradient_like(rows, cols, 50), rnd((rows, cols), 52), torch.zeros(rows, cols, device="cuda"),
                         rnd((rows, cols), 53) * 1e37, rnd((rows, cols), 54) * 1e-4])
        got = nz.orthogonalize(g)
        for i in (0, 1, 3, 4):
            assert torch.equal(got[i], nz.orthogonalize(g[i]))
            assert _rel(got[i], _ortho_ref(g[i])) <= ORTHO_TOL
        assert torch.equal(got[2], torch.zeros_like(got[2]))
        for extra, offset in ((1, 0), (4, 0), (4, 1)):
            out = padded(torch.zeros(rows, cols, device="cuda"), extra, offset)
            before = out._base.clone()
            nz.orthogonalize(padded(g[0], extra, offset), out=out)
            assert torch.equal(out, got[0])
            out.zero_()
            assert torch.equal(out._base, before)
        assert torch.equal(nz.orthogonalize(g[::2]), got[::2])
        # a norm beyond fp32's largest number, and one of subnormal numbers (without eps); in place
        huge, tiny = g[1].sign() * 3e38, g[1] * 1e-41
        assert _rel(nz.orthogonalize(huge), _ortho_ref(huge)) <= ORTHO_TOL
        assert _rel(nz.orthogonalize(tiny, eps=0.0), _ortho_ref(tiny, eps=0.0)) <= ORTHO_TOL
        assert torch.equal(nz.orthogonalize(torch.zeros_like(tiny), eps=0.0), torch.zeros_like(tiny))
        inplace = g[0].clone()
        assert nz.orthogonalize(inplace, out=inplace) is inplace and torch.equal(inplace, got[0])
        bad = g.clone()
        bad[1, 2, 3] = math.nan
        got2 = nz.orthogonalize(bad)
        assert torch.isnan(got2[1]).any() and torch.equal(got2[0], got[0]) and torch.equal(got2[3], got[3])
    assert nz.orthogonalize(torch.empty(0, 5, device="cuda")).shape == (0, 5)
    assert nz.orthogonalize(torch.empty(2, 0, 5, device="cuda")).shape == (2, 0, 5)
    assert nz.device_status() == 0


@pytest.mark.parametrize("shape", [(60, 100), (100, 60), (3, 70, 40), (1, 1)])
@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_step(shape, nesterov):
    w, m, g = rnd(shape, 60), rnd(shape, 61), rnd(shape, 62)
    lr, mu, wd = 0.02, 0.9, 0.1
    m2 = mu * m.double() + g.double()
    u = g.double() + mu * m2 if nesterov else m2
    rows, cols = shape[-2:]
    o = torch.stack([_ortho_ref(x) for x in u.reshape(-1, rows, cols)]).reshape(shape)
    step = lr * max(1.0, rows / cols) ** 0.5
    want = (1 - lr * wd) * w.double() - step * o
    got_w, got_m = w.clone(), m.clone()
    assert nz.muon_step(got_w, got_m, g, lr, mu=mu, weight_decay=wd, nesterov=nesterov) is got_w
    within(got_m, m2, 2 * U * (m.abs() + g.abs()))
    err = torch.linalg.norm(got_w.double() - want)
    assert err <= step * ORTHO_TOL * torch.linalg.norm(o) + 4 * U * torch.linalg.norm(w)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_logprob_of_a_largest_number(dtype):
    """A token forced by the type's largest number takes all of the probability; two of them share it."""
    big = torch.finfo(dtype).max
    x = rnd((4, 3001), 70, dtype)
    x[0, 7] = big
    x[1, 7] = x[1, 2900] = big
    x[2, :] = -math.inf
    x[2, 2000] = big
    t = torch.tensor([7, 2900, 2000, 0], device="cuda")
    f = nz.token_logprobs(x, t, top_k=2)
    ln2 = math.log(2.0)
    within(f.logprob[:3], torch.tensor([0.0, -ln2, 0.0], device="cuda"), 2 * U)
    within(f.entropy[:3], torch.tensor([0.0, ln2, 0.0], device="cuda"), 2 * U)
    assert f.top_index[:3, 0].tolist() == [7, 7, 2000] and f.top_index[1, 1] == 2900


# ---- all of them together ----------------------------------------------------------------------------------
def _token_model(p, idx, targets):
    """Rows of a table, layer norm, Linear, log probability of the next token: forward and backward by this library."""
    e = nz.embedding(p["table"], idx, scale=2.0)
    h, mean, rstd = nz.layernorm_forward(e, p["gamma"], p["beta"])
    logits = nz.linear_forward(h, p["w"])
    f = nz.token_logprobs(logits, targets, top_k=3)
    n = idx.numel()
    dlogits = nz.token_logprobs_backward(logits, targets, f.lse, f.entropy, torch.full((n,), -1.0 / n, device="cuda"))
    d = {k: torch.zeros_like(v) for k, v in p.items()}
    dh = torch.zeros_like(h)
    nz.linear_backward(h, p["w"], None, dlogits, dx=dh, dw=d["w"])
    de = torch.empty_like(e)
    nz.layernorm_backward(dh, e, mean, rstd, p["gamma"], de, d["gamma"], d["beta"], overwrite_dx=True)
    nz.embedding_backward(de, idx, d["table"], scale=2.0)
    return f, d


def test_token_model_training_step():
    vocab, dim, n = 501, 96, 70
    p = {"table": rnd((vocab, dim), 70), "gamma": rnd((dim,), 71) * 0.1 + 1, "beta": rnd((dim,), 72) * 0.1,
         "w": rnd((vocab, dim), 73) * 0.1}
    g = torch.Generator("cuda").manual_seed(74)
    idx = torch.randint(0, vocab, (n,), device="cuda", generator=g)
    idx[10:20] = idx[0]
    targets = torch.randint(0, vocab, (n,), device="cuda", generator=g)
    f, d = _token_model(p, idx, targets)
    q = {k: v.double().requires_grad_() for k, v in p.items()}
    e = q["table"][idx] * 2.0
    h = torch.nn.functional.layer_norm(e, (dim,), q["gamma"], q["beta"], 1e-5)
    logits = h @ q["w"].mT
    loss = torch.nn.functional.cross_entropy(logits, targets)
    loss.backward()
    # Linear rounds its operands to fp16 (2^-11 a product, two products in a chain): logits near 1 off by 2^-11 at most
    assert abs(float(-f.logprob.double().mean() - loss.detach())) <= 2.0 ** -10
    for k in p:
        assert _rel(d[k], q[k].grad) <= 4 * 2.0 ** -11, k
    # the update: the matrix by Muon, the vectors by plain descent; the loss is computed again on the new weights
    momentum = torch.zeros_like(p["w"])
    nz.muon_step(p["w"], momentum, d["w"], lr=0.01)
    assert torch.equal(momentum, d["w"]) and torch.isfinite(p["w"]).all()
    f2, _ = _token_model(p, idx, targets)
    assert torch.isfinite(f2.logprob).all()
    assert nz.device_status() == 0


def test_captured_step_equals_eager():
    vocab, dim, n = 300, 64, 40
    p = {"table": rnd((vocab, dim), 80), "gamma": rnd((dim,), 81) * 0.1 + 1, "beta": rnd((dim,), 82) * 0.1, "w": rnd((vocab, dim), 83) * 0.1}
    idx = torch.randint(0, vocab, (n,), device="cuda", generator=torch.Generator("cuda").manual_seed(84))
    targets = idx.roll(-1).contiguous()
    run = lambda: (_token_model(p, idx, targets), nz.orthogonalize(p["w"]))
    (f0, d0), o0 = run()
    graphs = []
    side = torch.cuda.Stream()
    for _ in range(2):  # two graphs side by side: their scratch is their own
        with torch.cuda.stream(side):
            run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        graphs.append((graph, out))
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(a):
            graphs[0][0].replay()
        with torch.cuda.stream(b):
            graphs[1][0].replay()
    torch.cuda.synchronize()
    for _, ((f, d), o) in graphs:
        assert all(torch.equal(x, y) for x, y in zip(f, f0)) and torch.equal(o, o0)
        # Linear's weight gradient may be shared among CTAs with atomics; the others are the same bits
        assert all(torch.equal(d[k], d0[k]) for k in ("gamma", "beta", "table"))
    idx.copy_(idx.flip(0))
    targets.copy_(idx.roll(-1))
    (f0, d0), _ = run()
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1][0][0].logprob, f0.logprob) and torch.equal(graphs[0][1][0][1]["table"], d0["table"])


def test_calls_on_several_streams():
    xs = [rnd((200 + 50 * i, 300), 90 + i) for i in range(4)]
    g = [rnd((150, 200 + 10 * i), 95 + i) for i in range(4)]
    idx = [torch.randint(0, 70, (5000,), device="cuda", generator=torch.Generator("cuda").manual_seed(99 + i)) for i in range(4)]
    dy = rnd((5000, 40), 103)
    one = lambda i: (nz.layernorm_forward(xs[i]), nz.orthogonalize(g[i]), nz.token_logprobs(xs[i], idx[i][: xs[i].shape[0]], top_k=4),
                     nz.embedding_backward(dy, idx[i], torch.empty(70, 40, device="cuda"), overwrite=True))
    want = [one(i) for i in range(4)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for _ in range(3):
        got = []
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append(one(i))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a[0], b[0])) and torch.equal(a[1], b[1])
        assert all(torch.equal(x, y) for x, y in zip(a[2], b[2])) and torch.equal(a[3], b[3])


def test_far_offsets():
    """Rows whose elements lie beyond 2^31 elements of their tensor's start."""
    vocab, dim = 70000, 32776  # 2.3e9 elements
    table = torch.empty(vocab, dim, dtype=F16, device="cuda")
    table[-2:] = rnd((2, dim), 110, F16)
    idx = torch.tensor([vocab - 1, vocab - 2, vocab - 1], device="cuda")
    assert torch.equal(nz.embedding(table, idx), table[idx])
    view = table[:, :1000]
    view[-3:] = rnd((3, 1000), 111, F16)
    t = torch.arange(vocab, device="cuda") % 1000
    f = nz.token_logprobs(view[-3:], t[-3:], top_k=4)
    view[:-3] = 0
    whole = nz.token_logprobs(view, t, top_k=4)
    assert torch.equal(whole.logprob[-3:], f.logprob) and torch.equal(whole.top_index[-3:], f.top_index)
    y, mean, rstd = nz.layernorm_forward(view)
    assert torch.equal(y[-3:], nz.layernorm_forward(view[-3:])[0])
    nz.layernorm_forward(view, out=view)
    assert torch.equal(view[-3:], y[-3:])


def test_command_line_runs_every_operator():
    import json
    import subprocess
    import sys
    r = subprocess.run([sys.executable, "-m", "neuzephyr_b200", "tokens", "100", "500", "96", "--dtype", "f16"],
                       capture_output=True, text=True, timeout=300,
                       cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert r.returncode == 0, r.stderr[-2000:]
    line = json.loads(r.stdout.splitlines()[-1])
    assert line["status"] == 0 and len(line["ms"]) == 7 and all(ms > 0 for ms in line["ms"].values())


def test_captured_behind_copies_and_other_streams():
    """The first kernel of a call is launched programmatically: in a graph it may follow a copy, a memset or another
    stream's work instead of a kernel."""
    src, other = rnd((96, 160), 90), rnd((96, 160), 91)
    g, cleared = torch.empty_like(src), torch.ones(4096, device="cuda")
    idx = torch.arange(50, device="cuda")
    dtable, dy = torch.empty((60, 32), device="cuda"), rnd((50, 32), 92)
    side = torch.cuda.Stream()

    def run():
        g.copy_(src)  # a copy right before
        a = nz.orthogonalize(g)
        cleared.zero_()  # a memset
        b = nz.orthogonalize(g)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            g.copy_(other)
        torch.cuda.current_stream().wait_stream(side)  # two streams join
        c = nz.orthogonalize(g)
        cleared.zero_()
        nz.embedding_backward(dy, idx, dtable, overwrite=True)
        return a, b, c

    want = [nz.orthogonalize(t) for t in (src, src, other)]
    assert all(torch.equal(x, y) for x, y in zip(run(), want))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for _ in range(3):
        for x in got:
            x.zero_()
        dtable.fill_(-1.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))
        assert torch.equal(dtable[:50], dy) and not dtable[50:].any()


# ---- rows at the border of fp32's range, whatever their length and alignment ---------------------------------
@pytest.mark.parametrize("dim", [9, 300, 301, 1000, 1024, 5003, 16000])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_layernorm_rows_of_large_numbers(dim, dtype):
    """What a thread holds beside its row (places without an element, neighbours in a cut block) must not reach the sums, not
    even as the square of a mean beyond 2^64 times zero."""
    x = torch.zeros(6, dim, device="cuda")
    x[0] = 2.0 ** 63
    x[1, 0] = x[2, -1] = 1.5e19  # squares 2.2e38, of which fp32 holds one
    x[3] = rnd((dim,), 120) * 1e17
    x[4, 0] = x[5, -1] = 1e38    # the sum fits, the squares do not: 1 / sqrt(inf)
    x = x.to(dtype)
    for v in (x, padded(x, 1), padded(x, 8, 1), padded(x, 3, 2)):
        for gamma, beta in ((None, None), (rnd((dim,), 121) + 1, rnd((dim,), 122))):
            y, mean, rstd = nz.layernorm_forward(v, gamma, beta)
            _check_norm(x[:4], gamma, beta, 1e-5, (y[:4], mean[:4], rstd[:4]))
            within(mean[4:], x[4:].double().mean(1), CHAIN * U * 1e38 / dim)
            assert torch.equal(rstd[4:], torch.zeros(2, device="cuda"))
            assert torch.equal(y[4:], torch.zeros_like(y[4:]) if beta is None else beta.to(dtype).expand(2, dim))


@pytest.mark.parametrize("dim", [9, 300, 301, 1000, 1024, 5003, 9001, 16000])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_layernorm_backward_rows_of_large_numbers(dim, dtype):
    """A mean whose product with rstd leaves fp32's range, beside places that hold no element of the row."""
    rows = 5
    x = torch.full((rows, dim), 2.0 ** 122, device="cuda").to(dtype)
    mean, rstd = torch.full((rows,), 2.0 ** 122, device="cuda"), torch.full((rows,), 316.25, device="cuda")
    dy, gamma = rnd((rows, dim), 123, dtype), rnd((dim,), 124) + 1
    for gm in (gamma, None):
        g = dy.double() * (1.0 if gm is None else gm.double())
        want = 316.25 * (g - g.mean(1, keepdim=True))  # h is 0
        tol = 316.25 * (g.abs() + g.abs().mean(1, keepdim=True)) * 2 * CHAIN * U
        for extra, offset in ((0, 0), (1, 0), (8, 1)):
            dx = padded(torch.zeros_like(x), extra, offset)
            dg, db = torch.full((dim,), math.nan, device="cuda"), torch.full((dim,), math.nan, device="cuda")
            nz.layernorm_backward(padded(dy, extra, offset), padded(x, extra, offset), mean, rstd, gm, dx, dg, db, overwrite_dx=True,
                                  overwrite_dparams=True)
            within(dx, want, tol + half_step(dtype) * (want.abs() + tol))
            assert torch.equal(dg, torch.zeros_like(dg))
            within(db, dy.double().sum(0), dy.double().abs().sum(0) * (rows + 32) * U)


def test_layernorm_of_rows_without_elements():
    torch.full((64,), 5.0, device="cuda")  # what the allocator hands out next is not NaN by chance
    y, mean, rstd = nz.layernorm_forward(torch.empty(3, 0, device="cuda"))
    assert y.shape == (3, 0) and torch.isnan(mean).all() and torch.isnan(rstd).all()
    dx, none = torch.empty(3, 0, device="cuda"), torch.empty(0, device="cuda")
    nz.layernorm_backward(y, y, mean, rstd, none, dx, none, none, overwrite_dx=True, overwrite_dparams=True)


# ---- many rows: several groups to a CTA that walk different numbers of rows, joined at the end -----------------
@pytest.mark.parametrize("rows,dim", [(1500, 96), (3001, 1027), (5000, 216), (2500, 5003), (9500, 2048), (40001, 33)])
@pytest.mark.parametrize("dtype", TYPES)
def test_layernorm_forward_of_many_rows(rows, dim, dtype):
    test_layernorm_forward(rows, dim, dtype)


@pytest.mark.parametrize("rows,dim", [(2500, 1027), (5000, 216), (9500, 2048), (3000, 5003), (1777, 9000), (40001, 33)])
@pytest.mark.parametrize("dtype", TYPES)
def test_layernorm_backward_of_many_rows(rows, dim, dtype):
    test_layernorm_backward(rows, dim, dtype)


# ---- tables above 2^23 elements and more than 2048 tokens: rows cleared beside the sort, by the marks ----------
@pytest.mark.parametrize("tokens,vocab,dim", [(2049, 70001, 131), (5000, 70001, 131), (16384, 40000, 256), (40000, 60000, 200)])
@pytest.mark.parametrize("dtype", TYPES)
def test_embedding_backward_of_large_tables(tokens, vocab, dim, dtype):
    test_embedding_backward(tokens, vocab, dim, dtype)


def test_embedding_backward_of_large_tables_strides():
    tokens, vocab, dim = 20000, 70001, 131
    g = torch.Generator("cuda").manual_seed(125)
    idx = torch.randint(0, vocab, (tokens,), device="cuda", generator=g)
    idx[::3] = 70000  # a third of the text is the table's last row
    dy = rnd((tokens, dim), 126, BF16)
    plain = torch.full((vocab, dim), math.nan, device="cuda")
    nz.embedding_backward(dy, idx, plain, overwrite=True)
    want, mags, count = _embedding_grad(dy, idx, vocab, 1.0, None)
    within(plain, want, mags * (count + 6) * U + 1e-30)
    for extra, offset in ((1, 0), (5, 3), (13, 1)):
        out = padded(torch.full((vocab, dim), math.nan, device="cuda"), extra, offset)
        nz.embedding_backward(dy, idx, out, overwrite=True)
        assert torch.equal(out, plain)
        out.fill_(77.0)
        assert (out._base == 77.0).all()  # nothing between the rows was written


# ---- large sides: 256 x 256 tiles by pairs of CTAs in all three products, with remainders ----------------------
def _tiles_launched(run):
    """Which tiles (pair of CTAs?, columns, product) a call launches, by the kernels' names; None where no profiler runs."""
    import re
    from torch.profiler import ProfilerActivity, profile
    with profile(activities=[ProfilerActivity.CUDA]) as p:
        run()
        torch.cuda.synchronize()
    if not any(e.device_type == torch.autograd.DeviceType.CUDA for e in p.events()):
        return None
    names = {e.name for e in p.events() if "ns_product_kernel" in e.name}
    found = {re.search(r"NsCfg<\(?(?:bool\))?(\w+), ?(?:\(int\))?(\d+)>, ?(?:\(int\))?(\d+)", n) for n in names}
    assert None not in found, names
    return {(m[1] in ("true", "1"), int(m[2]), int(m[3])) for m in found}


@pytest.mark.parametrize("batch,rows,cols", [(1, 2103, 2331), (1, 2331, 2103), (3, 2049, 2600), (2, 2600, 2049), (1, 4103, 4500), (1, 4500, 4103)])
def test_orthogonalize_by_pairs(batch, rows, cols):
    g = torch.stack([_gradient_like(rows, cols, 130 + i) for i in range(batch)])
    got = nz.orthogonalize(g)
    for i in range(batch):
        assert _rel(got[i], _ortho_ref(g[i])) <= ORTHO_TOL
    assert torch.equal(got, nz.orthogonalize(g))
    half = nz.orthogonalize(g.to(BF16), out_dtype=F16)
    assert _rel(half[0], _ortho_ref(g[0].to(BF16))) <= ORTHO_TOL + half_step(F16)
    assert _tiles_launched(lambda: nz.orthogonalize(g)) in (None, {(True, 256, mode) for mode in range(3)})
    assert nz.device_status() == 0


@pytest.mark.parametrize("shape", [(2103, 2331), (2331, 2103)])
def test_muon_step_by_pairs(shape):
    w, m, g = rnd(shape, 140), rnd(shape, 141), rnd(shape, 142)
    got_w, got_m = w.clone(), m.clone()
    nz.muon_step(got_w, got_m, g, 0.02, mu=0.9, weight_decay=0.1)
    m2 = 0.9 * m.double() + g.double()
    o = _ortho_ref(g.double() + 0.9 * m2)
    step = 0.02 * max(1.0, shape[0] / shape[1]) ** 0.5
    err = torch.linalg.norm(got_w.double() - ((1 - 0.02 * 0.1) * w.double() - step * o))
    assert err <= step * ORTHO_TOL * torch.linalg.norm(o) + 4 * U * torch.linalg.norm(w)
    within(got_m, m2, 2 * U * (m.abs() + g.abs()))


FIRST_CALL = """
import torch
import neuzephyr_b200 as nz
x, t = torch.randn(70, 300, device="cuda"), torch.randint(0, 300, (70,), device="cuda")
table, dy, idx = torch.empty(70001, 131, device="cuda"), torch.randn(5000, 131, device="cuda"), torch.randint(0, 70001, (5000,), device="cuda")
run = {"embedding": lambda: nz.embedding(x, t % 70), "embedding_backward": lambda: nz.embedding_backward(dy, idx, table, overwrite=True),
       "layernorm": lambda: nz.layernorm_forward(x)[0], "token_logprobs": lambda: nz.token_logprobs(x, t, top_k=3).logprob,
       "orthogonalize": lambda: nz.orthogonalize(x)}["CALL"]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = run()
graph.replay()
torch.cuda.synchronize()
replayed = y.clone()
assert torch.equal(replayed, run())
"""


@pytest.mark.parametrize("call", ["embedding", "embedding_backward", "layernorm", "token_logprobs", "orthogonalize"])
def test_first_call_of_a_process_within_a_capture(call):
    import subprocess
    import sys
    r = subprocess.run([sys.executable, "-c", FIRST_CALL.replace("CALL", call)], capture_output=True, text=True, timeout=300,
                       cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert r.returncode == 0, r.stderr[-2000:]


# ---- products of 22-bit operands ------------------------------------------------------------------------------
def _uneven_outer(rows, cols, seed):
    """Rank one, entries whose sizes differ by orders of magnitude: a gradient of one token with outlying features."""
    u, v = (rnd((rows,), seed) * 2).exp(), (rnd((cols,), seed + 1) * 2).exp()
    return torch.outer(u, v * rnd((cols,), seed + 2).sign())


def _ortho_noise(rows, cols, low_rank):
    """Relative error: every sum of a product goes through at most 3 K / 16 + 8 additions that cut off up to 2 u (three terms,
    sixteen elements an addition, the epilogue), three products in each of five steps. In what a matrix of low rank leaves empty the
    noise of a step grows by 3.4445 in each later one, while the result stays near 1: 1 + 3.4445 + ... + 3.4445^4 = 198."""
    return (198 if low_rank else 5) * 3 * (3 * max(rows, cols) / 16 + 8) * 2 * U


@pytest.mark.parametrize("rows,cols", [(5, 144), (144, 5), (16, 64), (64, 96), (100, 300), (300, 100), (256, 512), (512, 256), (1000, 1400),
                                       (2331, 2103)])
@pytest.mark.parametrize("low_rank", [False, True])
def test_orthogonalize_keeps_what_fp32_holds(rows, cols, low_rank):
    tol = _ortho_noise(rows, cols, low_rank)
    if low_rank:
        cases = [torch.outer(rnd((rows,), 150), rnd((cols,), 151)), _uneven_outer(rows, cols, 152),
                 rnd((rows, 3), 155) @ rnd((3, cols), 156)]
    else:
        cases = [rnd((rows, cols), 157), _gradient_like(rows, cols, 158)]
    for g in cases:
        want = _ortho_ref(g)
        assert _rel(nz.orthogonalize(g), want) <= tol
        for out_dtype in (F16, BF16):
            assert _rel(nz.orthogonalize(g, out_dtype=out_dtype), want) <= tol + half_step(out_dtype)
        w, m = rnd((rows, cols), 160), torch.zeros(rows, cols, device="cuda")
        start = w.double()
        nz.muon_step(w, m, g, 0.5, scale=1.0, mu=0.0)
        err = torch.linalg.norm(w.double() - (start - 0.5 * want))
        assert err <= 0.5 * tol * torch.linalg.norm(want) + 4 * U * torch.linalg.norm(start)


def test_token_logprobs_are_rounded_as_few_times_as_they_need():
    """lse = top + ln sum: the logarithm's rounding and the addition's, each spread over half a step to either side (rms a step /
    sqrt(12)); a quarter more is allowed for the sum's own roundings and a logarithm that is off by up to a step."""
    rows, vocab = 4096, 2999
    x = rnd((rows, vocab), 170) * 0.3 - 2.0  # lse near 6 and ln sum near 7: steps of 2^-21
    f = nz.token_logprobs(x, torch.zeros(rows, dtype=torch.int64, device="cuda"))
    want = torch.logsumexp(x.double(), 1)
    assert want.min() > 4 and want.max() < 8
    rms = (f.lse.double() - want).square().mean().sqrt()
    assert rms <= 1.25 * math.sqrt(2 / 12) * 2.0 ** -21
