"""Categorical observations: token log probabilities, entropy, top alternatives, the 'categorical' likelihood of the ELBO
loss and distillation from a teacher's top logits, against plain float64 on the CPU.

Tolerances.  A float32 statistic of a row: each exponential is off by the rounding of (x - m) log2(e) (half a step of a
number of at most 2^6 = 64 where 2^-64 still counts: 2^-19 in absolute terms, weighted by an exponential that has then
long decayed; for the terms that carry the sum it is below 2^-21) plus an ulp of v_exp_f32; a sum of V <= 2^18 terms in
256+ partial sums adds at most (V / 256 + 18) 2^-24.  ln s is then off by less than 2^-19 = 2e-6 absolutely, a log prob
by that plus 2^-24 of its size, the entropy by that times its weight |d| < 64.  So: log prob atol 4e-6 rtol 1e-6;
entropy and KL atol 2e-5.  Gradients: p is relative 4e-6 off (the same bound on ln p), the result is rounded once to its
type: half a step, torch.finfo(t).eps / 2 of the value."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
HALF = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def ref_rows(z):
    """float64 log softmax with the empty-row convention (-inf everywhere), and the entropy."""
    m = z.amax(-1, keepdim=True)
    empty = m == float('-inf')
    d = z - torch.where(empty, torch.zeros_like(m), m)
    s = d.exp().sum(-1, keepdim=True)
    logp = torch.where(empty, torch.full_like(d, float('-inf')), d - s.log())
    p = logp.exp()
    h = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(-1)
    return logp, p, h


def ref_top(z, k):
    """ids by value, ties by the lower index"""
    ids = torch.sort(z, dim=-1, descending=True, stable=True)[1]
    return ids[..., :k]


def close(a, b, rtol, atol):
    torch.testing.assert_close(a.detach().double().cpu(), b, rtol=rtol, atol=atol, equal_nan=True)


def check_grad(g, ref, scale):
    """`scale`: the size of the upstream factors, for the elements whose terms cancel."""
    r = HALF[g.dtype] + 6e-6
    atol = 2e-6 * scale + (2.0 ** -25 if g.dtype == torch.float16 else 0.0)   # half a step of fp16's subnormals
    torch.testing.assert_close(g.double().cpu(), ref, rtol=r, atol=atol, equal_nan=True)


def make(N, V, dt, seed, scale=3.0, stride=None, offset=0):
    """[N, V] logits on the GPU, as a view with a row stride / first element of its own, and their float64 values."""
    z = (torch.randn(N, V, generator=gen(seed)) * scale).to(TYPES[dt])
    stride = V if stride is None else stride
    base = torch.full((max(N - 1, 0) * stride + V + offset + 8,), float('nan'), dtype=TYPES[dt], device=DEV)
    view = base.as_strided((N, V), (stride, 1), offset)
    view.copy_(z.to(DEV))
    return view, z.double()


SHAPES = [(1, 1), (3, 2), (5, 7), (2, 63), (4, 64), (3, 65), (33, 256), (70, 257), (9, 511), (5, 512), (6, 1000), (3, 1024),
          (4, 2047), (2, 2048), (3, 2049), (5, 4097), (2, 8191), (2, 16384), (1, 20000), (3, 32768), (2, 50021), (1, 131072),
          (2, 200003)]


@pytest.mark.parametrize('dt', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('N,V', SHAPES)
def test_log_probs_entropy_and_alternatives(N, V, dt):
    from vae_amd import functional as F_
    x, z = make(N, V, dt, 7 * N + V)
    tok = torch.randint(0, V, (N,), generator=gen(V))
    k = min(V, 9)
    lp, h, top, ids = F_.token_log_probs(x, tok.to(DEV), top_k=k)
    logp, _, hr = ref_rows(z)
    close(lp, logp.gather(1, tok[:, None])[:, 0], 1e-6, 4e-6)
    close(h, hr, 1e-6, 2e-5)
    want = ref_top(z, k)
    assert torch.equal(ids.cpu(), want)
    close(top, logp.gather(1, want), 1e-6, 4e-6)
    lp2, h2, top2, ids2 = F_.token_log_probs(x, tok.to(torch.int32).to(DEV), want_entropy=False)
    assert h2 is None and top2 is None and ids2 is None
    close(lp2, logp.gather(1, tok[:, None])[:, 0], 1e-6, 4e-6)


@pytest.mark.parametrize('dt', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('V', [64, 300, 4096, 40000])
@pytest.mark.parametrize('k', [1, 2, 20, 64])
def test_alternatives_with_ties(V, k, dt):
    """Few distinct values: nearly every comparison is a tie; and rows of one value."""
    from vae_amd import functional as F_
    z = torch.randint(-2, 3, (4, V), generator=gen(V + k)).double()
    z[1] = 1.5
    z[2] = torch.arange(V).flip(0).double() // 7 % 100
    z[3] = torch.arange(V).double() // 5 % 90
    z[0, ::2] *= -0.0 if V == 64 else 1.0          # +0 and -0 are one value
    x = z.to(TYPES[dt]).to(DEV)
    _, _, top, ids = F_.token_log_probs(x, top_k=k)
    assert torch.equal(ids.cpu(), ref_top(z, k))
    close(top, ref_rows(z)[0].gather(1, ids.cpu()), 1e-6, 4e-6)


@pytest.mark.parametrize('dt', ['f32', 'bf16'])
@pytest.mark.parametrize('V,k', [(40, 40), (64, 64), (2100, 64), (70000, 24)])
def test_alternatives_that_sit_badly(V, k, dt):
    """The large values all where one thread (or one block of a split row) reads them: a stride of 256 vectors, the row's
    start, its end."""
    from vae_amd import functional as F_
    vec = 4 if dt == 'f32' else 8
    z = torch.randn(4, V, generator=gen(V)).to(TYPES[dt]).double()
    big = torch.arange(min(V, 200)).double() * 0.5 + 20
    z[0, :big.numel()] = big
    z[1, V - big.numel():] = big.flip(0)
    col = torch.arange(0, V, 256 * vec)
    for i in range(vec):
        c = col + i
        c = c[c < V]
        z[2, c] = 30.0 + torch.arange(c.numel()).double() * 0.25 + i
    z[3] = torch.sort(z[3])[0]
    z = z.to(TYPES[dt]).double()
    _, _, top, ids = F_.token_log_probs(z.to(TYPES[dt]).to(DEV), top_k=k)
    assert torch.equal(ids.cpu(), ref_top(z, k))


@pytest.mark.parametrize('dt', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('V', [31, 256, 1500, 30000])
def test_masks_and_extremes(V, dt):
    """-inf masks down to one and to no entry, the type's lowest value as a mask (a whole row of it too), its largest
    value, very negative rows, +inf and NaN."""
    from vae_amd import functional as F_
    low, high = torch.finfo(TYPES[dt]).min, torch.finfo(TYPES[dt]).max
    z = torch.randn(12, V, generator=gen(V)).to(TYPES[dt]).double()
    z[0, :] = float('-inf'); z[0, V // 2] = 1.0
    z[1, :] = float('-inf')
    z[2, :] = low; z[2, 3] = 0.5
    z[3, :] = low
    z[4, :] = low; z[4, 5] = float('-inf')
    z[5, 7] = high
    z[6, :] -= 30000.0
    z[7, ::2] = float('-inf')
    z[8, 2] = float('inf')
    z[9, 4] = float('nan')
    z[10, :] = high
    z[11, :] = float('-inf'); z[11, 1] = low
    z = z.to(TYPES[dt]).double()
    tok = torch.tensor([V // 2, 3, 3, 9, 9, 7, 11, 1, 2, 4, 6, 1])
    k = 20
    x = z.to(TYPES[dt]).to(DEV).requires_grad_(True)
    lp, h, top, ids = F_.token_log_probs(x, tok.to(DEV), top_k=k)
    logp, p, hr = ref_rows(z)
    bad = torch.tensor([8, 9])
    fine = torch.tensor([i for i in range(12) if i not in (8, 9)])
    want = logp.gather(1, tok[:, None])[:, 0]
    close(lp[fine.to(DEV)], want[fine], 1e-6, 4e-6)
    close(h[fine.to(DEV)], hr[fine], 1e-6, 2e-5)
    assert torch.equal(ids.cpu()[fine], ref_top(z, k)[fine])
    close(top[fine.to(DEV)], logp.gather(1, ref_top(z, k))[fine], 1e-6, 4e-6)
    assert bool(torch.isnan(lp[bad.to(DEV)]).all()) and bool(torch.isnan(h[bad.to(DEV)]).all())
    assert bool(torch.isnan(top[bad.to(DEV)]).all())
    idb = ids.cpu()[bad]
    assert bool(((idb >= -1) & (idb < V)).all())
    ga, gh = torch.randn(12, generator=gen(1)), torch.randn(12, generator=gen(2))
    g, = torch.autograd.grad([lp, h], [x], [ga.to(DEV), gh.to(DEV)])
    plogp = torch.where(p > 0, p * logp, torch.zeros_like(p))
    ref = -ga.double()[:, None] * p - gh.double()[:, None] * (plogp + p * hr[:, None])
    ref[torch.arange(12), tok] += ga.double()
    ref[1] = 0.0                                    # no distribution, no gradient
    check_grad(g.cpu()[fine], ref[fine], 3.0)
    assert bool(torch.isnan(g.cpu()[bad]).all())


@pytest.mark.parametrize('dt', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('N,V,stride,offset', [(5, 100, 128, 0), (5, 100, 101, 3), (3, 1000, 1003, 1), (4, 4096, 4104, 8),
                                               (3, 4096, 4096, 1), (2, 30001, 30001, 5), (3, 30001, 30728, 0),
                                               (9, 256, 256, 2), (5, 255, 255, 1)])
def test_strides_and_alignment(N, V, stride, offset, dt):
    """Rows at any stride and any first element, NaN between them: nothing outside a row counts; the gradient is whole."""
    from vae_amd import functional as F_
    x, z = make(N, V, dt, V + offset, stride=stride, offset=offset)
    tok = torch.randint(0, V, (N,), generator=gen(3))
    tok[0], tok[-1] = 0, V - 1
    x.requires_grad_(True)
    lp, h, top, ids = F_.token_log_probs(x, tok.to(DEV), top_k=5)
    logp, p, hr = ref_rows(z)
    close(lp, logp.gather(1, tok[:, None])[:, 0], 1e-6, 4e-6)
    close(h, hr, 1e-6, 2e-5)
    assert torch.equal(ids.cpu(), ref_top(z, 5))
    ga, gh = torch.randn(N, generator=gen(1)), torch.randn(N, generator=gen(2))
    gt = torch.randn(N, 5, generator=gen(4))
    g, = torch.autograd.grad([lp, h, top], [x], [ga.to(DEV), gh.to(DEV), gt.to(DEV)])
    ref = -(ga.double() + gt.double().sum(1))[:, None] * p - gh.double()[:, None] * p * (logp + hr[:, None])
    ref[torch.arange(N), tok] += ga.double()
    ref.scatter_add_(1, ref_top(z, 5), gt.double())
    check_grad(g, ref, 8.0)
    kl, mean = F_.distill_top_logits(x, top.detach(), ids)
    assert kl.shape == (N,) and bool(torch.isfinite(mean))
    gm, = torch.autograd.grad(mean, x)
    q = torch.softmax(top.detach().double().cpu(), -1)
    refd = p.clone()
    refd.scatter_add_(1, ids.cpu(), -q)
    check_grad(gm, refd / N, 2.0 / N)


@pytest.mark.parametrize('dt', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('N,V', [(1, 1), (4, 3), (130, 256), (20, 1024), (7, 2049), (5, 16384), (3, 32768), (2, 65536),
                                 (2, 70001), (2, 131072), (1, 140000)])
@pytest.mark.parametrize('what', ['logp', 'entropy', 'both'])
def test_gradients(N, V, dt, what):
    from vae_amd import functional as F_
    x, z = make(N, V, dt, V, scale=2.0)
    x.requires_grad_(True)
    tok = torch.randint(0, V, (N,), generator=gen(V))
    ga, gh = torch.randn(N, generator=gen(1)), torch.randn(N, generator=gen(2))
    lp, h, _, _ = F_.token_log_probs(x, tok.to(DEV), want_entropy=what != 'logp')
    logp, p, hr = ref_rows(z)
    a = ga.double() if what != 'entropy' else torch.zeros(N).double()
    b = gh.double() if what != 'logp' else torch.zeros(N).double()
    outs = {'logp': [lp], 'entropy': [h], 'both': [lp, h]}[what]
    ups = {'logp': [ga], 'entropy': [gh], 'both': [ga, gh]}[what]
    g, = torch.autograd.grad(outs, [x], [u.to(DEV) for u in ups])
    ref = -a[:, None] * p - b[:, None] * p * (logp + hr[:, None])
    ref[torch.arange(N), tok] += a
    check_grad(g, ref, 6.0)


def test_gradient_against_differences():
    """Central differences of the forward kernels themselves, float32 (step 1e-2: truncation ~ step^2 = 1e-4 of a second
    derivative below 1, rounding 4e-6 / 1e-2)."""
    from vae_amd import functional as F_
    V, tok = 17, torch.tensor([4, -1, 16], device=DEV)
    x = torch.randn(3, V, generator=gen(0)).to(DEV)
    tl, ti = torch.randn(3, 3, generator=gen(1)).to(DEV), torch.tensor([[1, 5, 5], [-1, 2, 3], [0, 16, -1]], device=DEV)

    def value(v):
        lp, h, top, _ = F_.token_log_probs(v, tok, top_k=2)
        kl, _ = F_.distill_top_logits(v, tl, ti, temperature=1.7)
        # the padded row's alternatives are -inf by definition: left out
        return (0.7 * lp + 0.3 * h + 0.9 * kl).sum() + top[0].sum() + 0.5 * top[2].sum()

    xr = x.clone().requires_grad_(True)
    g, = torch.autograd.grad(value(xr), xr)
    step = 1e-2
    num = torch.zeros_like(x)
    for r in range(3):
        for j in range(V):
            d = torch.zeros_like(x)
            d[r, j] = step
            num[r, j] = (value(x + d) - value(x - d)) / (2 * step)
    torch.testing.assert_close(g, num, rtol=5e-3, atol=2e-3)


@pytest.mark.parametrize('V', [16, 256, 5000, 60000])
def test_padded_rows_are_not_read(V):
    """Rows behind a sequence's end hold NaN: they come out as padding says, gradients 0."""
    from vae_amd import functional as F_
    x = torch.randn(6, V, generator=gen(V)).to(DEV)
    x[2] = float('nan')
    x[5] = float('nan')
    tok = torch.tensor([0, V - 1, -100, 3, 1, -1], device=DEV)
    x.requires_grad_(True)
    lp, h, top, ids = F_.token_log_probs(x, tok, top_k=3)
    pad, live = [2, 5], [0, 1, 3, 4]
    assert bool((lp[pad] == 0).all()) and bool((h[pad] == 0).all())
    assert bool((ids[pad] == -1).all()) and bool((top[pad] == float('-inf')).all())
    assert bool(torch.isfinite(lp[live]).all()) and bool(torch.isfinite(h[live]).all())
    g, = torch.autograd.grad([lp, h], [x], [torch.ones_like(lp), torch.ones_like(h)], retain_graph=True)
    assert bool((g[pad] == 0).all()) and bool(torch.isfinite(g).all())
    g, = torch.autograd.grad(top[live].sum(), [x])
    assert bool((g[pad] == 0).all()) and bool(torch.isfinite(g).all())
    out = F_.nll(tok[:, None], x.detach()[:, None], 'categorical')
    assert bool((out[pad] == 0).all()) and bool(torch.isfinite(out).all())
    ids = torch.tensor([[0, 1]] * 6, device=DEV)
    ids[pad] = -1
    kl, mean = F_.distill_top_logits(x, torch.zeros(6, 2, device=DEV), ids, inv_count=0.25)
    assert bool((kl[pad] == 0).all()) and bool(torch.isfinite(mean))
    g, = torch.autograd.grad(mean, x)
    assert bool((g[pad] == 0).all()) and bool(torch.isfinite(g).all())


def test_ids_beyond_the_vocabulary_are_nan_not_reads():
    from vae_amd import functional as F_
    for V in (8, 300, 9000):
        x = torch.randn(3, V, generator=gen(V)).to(DEV).requires_grad_(True)
        tok = torch.tensor([1, V, 1 << 40], device=DEV)
        lp, h, _, _ = F_.token_log_probs(x, tok)
        assert bool(torch.isfinite(lp[0])) and bool(torch.isnan(lp[1:]).all()) and bool(torch.isfinite(h).all())
        g, = torch.autograd.grad(lp.sum(), x)
        assert bool(torch.isfinite(g[0]).all()) and bool(torch.isnan(g[1:]).all())
        out = F_.nll_elbo(tok[:, None], x[:, None], 'categorical', fuse_backward=True)
        g, = torch.autograd.grad(out[3][0], x)
        assert bool(torch.isfinite(g[0]).all()) and bool(torch.isnan(g[1:]).all())
        ids = torch.tensor([[0, 1], [2, V], [1 << 33, 0]], device=DEV)
        for fuse in (False, True):
            kl, mean = F_.distill_top_logits(x, torch.zeros(3, 2, device=DEV), ids, fuse_backward=fuse)
            assert bool(torch.isfinite(kl[0])) and bool(torch.isnan(kl[1:]).all())
            g, = torch.autograd.grad(mean, x)
            assert bool(torch.isfinite(g[0]).all()) and bool(torch.isnan(g[1:]).all())


# ---------------------------------------------------------------------------------------------------------------------
# the categorical likelihood of the ELBO loss
# ---------------------------------------------------------------------------------------------------------------------
def ref_elbo(z, x, kld, beta):
    B, V = z.shape[0], z.shape[-1]
    logp, p, _ = ref_rows(z.reshape(-1, V))
    tok = x.reshape(-1)
    live = tok >= 0
    lp = torch.where(live, logp.gather(1, tok.clamp(min=0)[:, None])[:, 0], torch.zeros(tok.numel()).double())
    nll = -lp.reshape(B, -1).sum(1)
    p = p.clone()
    p[torch.arange(tok.numel()), tok.clamp(min=0)] -= 1.0
    grad = (p * live[:, None]).reshape(z.shape)
    return nll, nll + beta * kld, nll + kld, grad


ELBO = [(1, (), 1), (4, (), 10), (3, (5,), 256), (6, (1, 4, 4), 256), (5, (3,), 1000), (4, (7,), 4096), (2, (3,), 30001),
        (2, (2,), 65536), (2, (1,), 131072), (1, (2,), 150000), (2, (4,), 20000)]


@pytest.mark.parametrize('dt', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('B,shape,V', ELBO)
@pytest.mark.parametrize('fuse', [True, False])
def test_loss_function_categorical(B, shape, V, dt, fuse):
    import vae_amd
    z = (torch.randn((B,) + shape + (V,), generator=gen(V)) * 2).to(TYPES[dt])
    x = torch.randint(0, V, (B,) + shape, generator=gen(B))
    if x.numel() > 2:
        x.view(-1)[1] = -100
    kld = (torch.rand(B, generator=gen(5)) * 4).to(TYPES[dt])
    xr = z.to(DEV).requires_grad_(True)
    kr = kld.to(DEV).requires_grad_(True)
    out = vae_amd.loss_function(xr, x.to(DEV), kr, 'categorical', kl_beta=0.5, fuse_backward=fuse)
    nll, loss, elbo, grad = ref_elbo(z.double(), x, kld.double(), 0.5)
    # nll is rounded to the type, then loss = nll + beta kld once more
    r = 2 * HALF[TYPES[dt]] + 2e-6
    close(out['loss'], loss, r, 1e-5)
    close(out['elbo'], elbo, r, 1e-5)
    close(out['loss_mean'], loss.mean(), 2 * r, 1e-5)
    close(out['nll_mean'], nll.mean(), 2 * r, 1e-5)
    close(out['kld_mean'], kld.double().mean(), 2 * r, 1e-5)
    g, gk = torch.autograd.grad(out['loss_mean'], [xr, kr])
    check_grad(g, grad / B, 1.0 / B)
    close(gk, torch.full((B,), 0.5 / B).double(), 2 * HALF[TYPES[dt]], 2.0 ** -25)


def test_loss_function_categorical_other_gradients():
    """A per-sample gradient, a mean gradient that is not 1, and a second backward of a kept graph, through the launch
    that has already stored d(loss_mean): the same as the two-pass form."""
    import vae_amd
    B, T, V = 5, 3, 700
    z = torch.randn(B, T, V, generator=gen(1))
    x = torch.randint(0, V, (B, T), generator=gen(2)).to(DEV)
    kld = torch.rand(B, generator=gen(3)).to(DEV)
    w = torch.rand(B, generator=gen(4)).to(DEV)
    got = {}
    for fuse in (True, False):
        xr = z.to(DEV).requires_grad_(True)
        out = vae_amd.loss_function(xr, x, kld, 'categorical', kl_beta=2.0, fuse_backward=fuse)
        got[fuse] = [torch.autograd.grad(3.0 * out['loss_mean'], xr, retain_graph=True)[0],
                     torch.autograd.grad(out['loss_mean'] + (w * out['elbo']).sum(), xr, retain_graph=True)[0],
                     torch.autograd.grad((w * out['loss']).sum(), xr, retain_graph=True)[0],
                     torch.autograd.grad(out['loss_mean'], xr)[0]]
    ref = ref_elbo(z.double(), x.cpu(), kld.double().cpu(), 2.0)[3]
    wd = w.double().cpu()[:, None, None]
    for a, b, r in zip(got[True], got[False], (3.0 / B * ref, (1.0 / B + wd) * ref, wd * ref, ref / B)):
        check_grad(a, r, 2.0)
        check_grad(b, r, 2.0)


def test_nll_forms_agree():
    """nll, the multi-sample form, the per-step form with its log-sum-exp, Autoencoder / VAENoKL and a host model's
    loss_function, all on the categorical likelihood."""
    import vae_amd
    from vae_amd import functional as F_
    B, T, V = 4, 3, 50
    zs = [torch.randn(B, T, V, generator=gen(i)) for i in range(3)]
    xs = [torch.randint(-1, V, (B, T), generator=gen(10 + i)) for i in range(3)]
    ref = [ref_elbo(z.double(), x, torch.zeros(B).double(), 1.0)[0] for z, x in zip(zs, xs)]
    d = lambda v: [t.to(DEV) for t in v]
    close(F_.nll(xs[0].to(DEV), zs[0].to(DEV), 'categorical'), ref[0], 1e-6, 1e-5)
    multi = [ref_elbo(z.double(), xs[0], torch.zeros(B).double(), 1.0)[0] for z in zs]
    close(F_.nll_multi_elbo(xs[0].to(DEV), d(zs), 'categorical')[0], sum(multi) / 3, 1e-6, 1e-5)
    kld = torch.rand(3 * B, generator=gen(9))
    out = F_.nll_steps_elbo(d(xs), d(zs), 'categorical', kld=kld.to(DEV), kl_beta=0.3, with_lse=True)
    nll = torch.cat(ref)
    close(out[0], nll, 1e-6, 1e-5)
    close(out[1], nll + 0.3 * kld.double(), 1e-6, 1e-5)
    close(out[3][0], (nll + 0.3 * kld.double()).mean(), 1e-6, 1e-5)
    close(out[6], torch.logsumexp((nll + kld.double()).view(3, B), 0), 1e-6, 1e-5)
    with pytest.raises(NotImplementedError):
        F_.nll_steps_elbo(d(xs), d(zs), 'categorical', kl_beta=[0.1, 0.2, 0.3])

    class Auto(vae_amd.AutoencoderMixin):
        config = {'nll_type': 'categorical'}

    xr = zs[0].to(DEV).requires_grad_(True)
    o = Auto().loss_function(xr, xs[0].to(DEV))
    close(o['loss_mean'], ref[0].mean(), 1e-6, 1e-5)
    g, = torch.autograd.grad(o['loss_mean'], xr)
    check_grad(g, ref_elbo(zs[0].double(), xs[0], torch.zeros(B).double(), 1.0)[3] / B, 1.0 / B)


@pytest.mark.parametrize('dt', ['bf16', 'f16'])
def test_forms_that_add_up_round_once(dt):
    """The multi-sample and the per-step form on 16-bit logits, with fp32 terms of the host's: every output is one rounding
    of the fp32 value (half a step), the gradients are whole."""
    from vae_amd import functional as F_
    B, T, V, S = 5, 4, 300, 3
    zs = [torch.randn(B, T, V, generator=gen(i)).to(TYPES[dt]) for i in range(S)]
    x = torch.randint(-1, V, (B, T), generator=gen(9))
    kld, add = torch.rand(B, generator=gen(1)) * 30, torch.rand(B, generator=gen(2))
    refs = [ref_elbo(z.double(), x, torch.zeros(B).double(), 1.0) for z in zs]
    half = HALF[TYPES[dt]]
    nll = sum(r[0] for r in refs) / S
    leaves = [z.to(DEV).requires_grad_(True) for z in zs]
    k = kld.to(DEV).requires_grad_(True)
    out = F_.nll_multi_elbo(x.to(DEV), leaves, 'categorical', kld=k, add=add.to(DEV), kl_beta=0.5)
    assert all(t.dtype == TYPES[dt] for t in out[:3])
    for got, want in zip(out, (nll, nll + add.double() + 0.5 * kld.double(), nll + kld.double())):
        close(got, want, half + 1e-6, 1e-5)
    close(out[3][:4], torch.stack([(nll + add.double() + 0.5 * kld.double()).mean(), (nll + kld.double()).mean(),
                                   nll.mean(), kld.double().mean()]), 1e-6, 1e-5)
    gs = torch.autograd.grad(out[3][0], leaves + [k])
    for g, r in zip(gs, refs):
        check_grad(g, r[3] / (B * S), 1.0 / (B * S))
    close(gs[-1], torch.full((B,), 0.5 / B).double(), 2.0 ** -22, 0.0)
    steps = F_.nll_steps_elbo([x.to(DEV)] * S, [z.to(DEV) for z in zs], 'categorical', kld=kld.repeat(S).to(DEV))
    per = torch.stack([r[0] + kld.double() for r in refs])
    close(steps[1], per.reshape(-1), half + 1e-6, 1e-5)
    close(steps[4], per.mean(0), half + 1e-6, 1e-5)
    with pytest.raises(ValueError):
        F_.nll_multi_elbo(x.to(DEV), leaves, 'categorical', kld=k[:2])
    with pytest.raises(ValueError):
        F_.nll_steps_elbo([x.to(DEV)] * S, [z.to(DEV) for z in zs], 'categorical', kld=k)


def test_vrnn_loss_over_categorical_steps():
    """VRNNMixin scores categorical steps one by one; a stateful annealer weighs every step by its own value."""
    from vae_amd.vrnn import VRNNMixin
    B, V, T = 3, 40, 4
    zs = [torch.randn(B, V, generator=gen(i)) for i in range(T)]
    xs = [torch.randint(0, V, (B,), generator=gen(20 + i)) for i in range(T)]
    klds = [torch.rand(B, generator=gen(30 + i)) for i in range(T)]

    class Host(VRNNMixin):
        config = {'nll_type': 'categorical', 'kl_beta': 1.0}
        reparameterizer = None
        calls = 0
        training = True

        def kld(self, dist):
            return dist['kld']

        def mut_info(self, dist, n):
            return None

        def compute_kl_beta(self, v):
            self.calls += 1
            return [v[0] * self.calls / T]

    leaves = [z.to(DEV).requires_grad_(True) for z in zs]
    out = Host().loss_function(leaves, [x.to(DEV) for x in xs], [{'kld': k.to(DEV)} for k in klds])
    want = sum(ref_elbo(z.double(), x, k.double(), (i + 1) / T)[1] for i, (z, x, k) in enumerate(zip(zs, xs, klds))) / T
    close(out['loss'], want, 1e-6, 1e-5)
    close(out['loss_mean'], want.mean(), 1e-6, 1e-5)
    gs = torch.autograd.grad(out['loss_mean'], leaves)
    for g, z, x, k in zip(gs, zs, xs, klds):
        check_grad(g, ref_elbo(z.double(), x, k.double(), 1.0)[3] / (B * T), 1.0 / B)


# ---------------------------------------------------------------------------------------------------------------------
# distillation
# ---------------------------------------------------------------------------------------------------------------------
def ref_distill(z, y, ids, tau):
    V = z.shape[1]
    logp, p, _ = ref_rows(z / tau)
    here = ids >= 0
    yy = torch.where(here, y / tau, torch.full_like(y, float('-inf')))
    logq, q, _ = ref_rows(yy)
    lp = logp.gather(1, ids.clamp(min=0))
    kl = torch.where(q > 0, q * (logq - lp), torch.zeros_like(q)).sum(1)
    some = (q.sum(1) > 0)
    grad = torch.where(some[:, None], p / tau, torch.zeros_like(p))
    grad.scatter_add_(1, ids.clamp(min=0), -q / tau)
    return kl, grad


DISTILL = [(1, 1, 1), (3, 8, 3), (5, 100, 7), (33, 256, 16), (4, 1000, 64), (6, 4097, 33), (2, 20000, 256), (3, 50021, 100),
           (2, 65536, 65), (2, 131072, 64), (1, 140001, 5)]


@pytest.mark.parametrize('dt,tdt', [('f32', 'f32'), ('bf16', 'f32'), ('bf16', 'bf16'), ('f16', 'f16')])
@pytest.mark.parametrize('N,V,K', DISTILL)
@pytest.mark.parametrize('tau', [1.0, 2.5])
def test_distillation(N, V, K, dt, tdt, tau):
    """Random ids (so some come twice), absent entries, both forms of the gradient."""
    from vae_amd import functional as F_
    z = (torch.randn(N, V, generator=gen(V)) * 2).to(TYPES[dt])
    y = (torch.randn(N, K, generator=gen(K)) * 3).to(TYPES[tdt])
    ids = torch.randint(0, V, (N, K), generator=gen(N))
    if K > 2:
        ids[:, 1] = ids[:, 0]
        ids[0, 2] = -1
        y[-1, 2] = float('-inf')
    if N > 2:
        ids[1] = -1
    kl_r, grad_r = ref_distill(z.double(), y.double(), ids, tau)
    for idt in (torch.int32, torch.int64):
        xr = z.to(DEV).requires_grad_(True)
        kl, mean = F_.distill_top_logits(xr, y.to(DEV), ids.to(idt).to(DEV), temperature=tau)
        close(kl, kl_r, 1e-6, 2e-5)
        close(mean, kl_r.mean(), 1e-6, 2e-5)
        g, = torch.autograd.grad(mean, xr, retain_graph=True)
        check_grad(g, grad_r / N, 2.0 / N)
        w = torch.rand(N, generator=gen(8))
        g, = torch.autograd.grad([kl, mean], [xr], [w.to(DEV), torch.tensor(0.5, device=DEV)])
        check_grad(g, (w.double()[:, None] + 0.5 / N) * grad_r, 2.0)
    with torch.no_grad():
        kl, _ = F_.distill_top_logits(z.to(DEV), y.to(DEV), ids.to(DEV), temperature=tau)
    close(kl, kl_r, 1e-6, 2e-5)


def test_distillation_scaled_mean_and_strided_teacher():
    from vae_amd import functional as F_
    N, V, K, tau = 6, 900, 10, 3.0
    z = torch.randn(N, V, generator=gen(1))
    big_y, big_i = torch.randn(N, 24, generator=gen(2)), torch.randint(0, V, (N, 24), generator=gen(3))
    y, ids = big_y[:, 3:3 + K], big_i[:, 5:5 + K]
    kl_r, grad_r = ref_distill(z.double(), y.double(), ids, tau)
    for up in (1.0, 128.0):
        xr = z.to(DEV).requires_grad_(True)
        kl, mean = F_.distill_top_logits(xr, big_y.to(DEV)[:, 3:3 + K], big_i.to(DEV)[:, 5:5 + K], temperature=tau,
                                         inv_count=tau * tau / N)
        close(kl, kl_r, 1e-6, 2e-5)
        close(mean, kl_r.mean() * tau * tau, 1e-6, 2e-4)
        g, = torch.autograd.grad(mean * up, xr)
        check_grad(g, grad_r * (tau * tau * up / N), 2.0 * up)


def test_distillation_masked_student_and_teacher_extremes():
    """A teacher entry whose student logit is masked: infinite KL, a finite gradient (p = 0 there); a teacher row of the
    type's lowest value is uniform; a masked student without teacher mass stays finite."""
    from vae_amd import functional as F_
    z = torch.randn(4, 60, generator=gen(1))
    z[0, 7] = float('-inf')
    z[1, 9] = float('-inf')
    z[3] = float('-inf')
    y = torch.randn(4, 3, generator=gen(2))
    y[2] = torch.finfo(torch.float32).min
    ids = torch.tensor([[7, 1, 2], [1, 2, 3], [4, 5, 6], [1, 2, 3]])
    xr = z.to(DEV).requires_grad_(True)
    kl, mean = F_.distill_top_logits(xr, y.to(DEV), ids.to(DEV))
    kl_r, grad_r = ref_distill(z.double(), y.double(), ids, 1.0)
    grad_r[3] = 0.0                                  # a student row of -inf: infinite KL, no gradient
    assert kl_r[0] == math.inf and kl_r[3] == math.inf
    close(kl, kl_r, 1e-6, 2e-5)
    g, = torch.autograd.grad(kl, xr, torch.ones(4, device=DEV))
    check_grad(g, grad_r, 2.0)


def test_losses_together_train():
    """A categorical decoder as it would be trained: token nll + KL of the latent + distillation from a teacher, one
    backward, the entropy read beside it; the gradient against float64."""
    import vae_amd
    from vae_amd import functional as F_
    B, T, V, K, tau = 4, 6, 500, 8, 2.0
    z = torch.randn(B, T, V, generator=gen(1))
    x = torch.randint(0, V, (B, T), generator=gen(2))
    x[1, 4:] = -1
    teacher = torch.randn(B, T, V, generator=gen(3))
    y, ids = teacher.topk(K, -1)
    ids = torch.where(x[..., None] < 0, torch.full_like(ids, -1), ids)
    xr = z.to(DEV).requires_grad_(True)
    kld = torch.rand(B, generator=gen(4)).to(DEV)
    dist = vae_amd.distillation(xr, y.to(DEV), ids.to(DEV), tau)
    _, ent, _, _ = F_.token_log_probs(xr, x.to(DEV))
    out = vae_amd.loss_function(xr, x.to(DEV), kld, 'categorical', kl_beta=0.5, extra_loss_terms={'distill': dist})
    loss = out['loss_mean'] - 0.01 * ent.sum()
    g, = torch.autograd.grad(loss, xr)
    zd = z.double().requires_grad_(True)
    live = x >= 0
    lp = torch.log_softmax(zd, -1)
    nll = -(lp.gather(2, x.clamp(min=0)[..., None])[..., 0] * live).sum(1)
    h = -(lp.exp() * lp).sum(-1) * live
    q = torch.softmax(y.double() / tau, -1)
    kl = ((q * (q.log() - torch.log_softmax(zd / tau, -1).gather(2, ids.clamp(min=0)))).sum(-1) * live).sum(1)
    ref = (nll + kl + 0.5 * kld.double().cpu()).mean() - 0.01 * h.sum()
    close(loss, ref.detach(), 1e-5, 1e-5)
    gr, = torch.autograd.grad(ref, zd)
    check_grad(g, gr, 1.0)


# ---------------------------------------------------------------------------------------------------------------------
# streams, graphs, refusals
# ---------------------------------------------------------------------------------------------------------------------
def _everything(x, tok, y, ids):
    from vae_amd import functional as F_
    lp, h, top, ti = F_.token_log_probs(x, tok, top_k=6)
    kl, mean = F_.distill_top_logits(x, y, ids, temperature=1.5)
    _, loss, _, means = F_.nll_elbo(tok[:, None], x[:, None], 'categorical', fuse_backward=True)
    g1, = torch.autograd.grad([lp, h], [x], [torch.ones_like(lp), torch.ones_like(h)])
    g2, = torch.autograd.grad(mean, x)
    g3, = torch.autograd.grad(means[0], x)
    return [t.detach() for t in (lp, h, top, ti, kl, mean, loss, means, g1, g2, g3)]


@pytest.mark.parametrize('N,V,dt', [(3, 200, 'f32'), (2, 40000, 'bf16'), (300, 5000, 'bf16')])
def test_repeats_streams_and_graphs_give_the_same_bits(N, V, dt):
    """Twice in a row, on a side stream, from a captured graph replayed between eager calls: equal bits each time."""
    import vae_amd
    x, _ = make(N, V, dt, 5)
    x = x.contiguous()
    tok = torch.randint(-1, V, (N,), generator=gen(1)).to(DEV)
    y, ids = torch.randn(N, 9, generator=gen(2)).to(DEV), torch.randint(0, V, (N, 9), generator=gen(3)).to(DEV)
    eager = _everything(x.clone().requires_grad_(True), tok, y, ids)
    for a, b in zip(eager, _everything(x.clone().requires_grad_(True), tok, y, ids)):
        assert torch.equal(a, b)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = _everything(x.clone().requires_grad_(True), tok, y, ids)
    torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(eager, side):
        assert torch.equal(a, b)
    static = x.clone()
    step = vae_amd.graph.capture(lambda: _everything(static.detach().requires_grad_(True), tok, y, ids))
    for turn in range(3):
        static.copy_(x if turn != 1 else x.flip(1))
        outs = step()
        want = eager if turn != 1 else _everything(x.flip(1).contiguous().requires_grad_(True), tok, y, ids)
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize('kind', ['nll', 'distill'])
def test_backward_captured_apart_from_its_forward(kind):
    """A stored gradient is multiplied in place: replays of a backward pass whose forward pass was eager must not
    multiply it again and again."""
    from vae_amd import functional as F_
    N, V = 12, 3000
    x = torch.randn(N, V, generator=gen(3)).to(DEV)
    tok = torch.randint(0, V, (N, 1), generator=gen(4)).to(DEV)
    y, ids = torch.randn(N, 5, generator=gen(5)).to(DEV), torch.randint(0, V, (N, 5), generator=gen(6)).to(DEV)

    def loss(x):
        if kind == 'nll':
            return F_.token_nll_elbo(tok, x[:, None], fuse_backward=True)[3][0]
        return F_.distill_top_logits(x, y, ids)[1]

    two = torch.full((), 2.0, device=DEV)
    xr = x.clone().requires_grad_(True)
    want, = torch.autograd.grad(loss(xr), xr, two)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        leaf = x.clone().requires_grad_(True)
        value = loss(leaf)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        g, = torch.autograd.grad(value, leaf, two)
    for _ in range(3):
        g.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        # the two forms round d, e = 2^d, the sum, 1 / s and the products apart.  p |d| < 0.6 (e^-y y at most 1/e) and p < 1
        # bound what each rounding moves: under 16 steps of 2^-24 of a gradient of 2 / N
        assert (g - want).abs().max() <= 16 * 2.0 ** -24 * 2.0 / N


@pytest.mark.parametrize('V', [40, 3000, 70000])
def test_an_id_beyond_the_vocabulary_in_a_masked_row(V):
    """Both at once: the id decides, in every form of the gradient."""
    from vae_amd import functional as F_
    x = torch.randn(3, V, generator=gen(1)).to(torch.bfloat16)
    x[1] = float('-inf')
    tok = torch.tensor([1, V, -1]).to(DEV)
    x = x.to(DEV)
    for fuse in (False, True):
        xr = x.clone().requires_grad_(True)
        out = F_.token_nll_elbo(tok[:, None], xr[:, None], fuse_backward=fuse)
        g, = torch.autograd.grad(out[3][0], xr)
        assert g[1].isnan().all() and (g[2] == 0).all() and not g[0].isnan().any()
        assert out[0][1].isnan() and out[0][2] == 0 and not torch.signbit(out[0][2])
    xr = x.clone().requires_grad_(True)
    lp, h, _, _ = F_.token_log_probs(xr, tok)
    g, = torch.autograd.grad(lp.sum() + h.sum(), xr)
    assert g[1].isnan().all() and (g[2] == 0).all() and not g[0].isnan().any()
    g, = torch.autograd.grad(F_.token_log_probs(xr, tok)[1].sum(), xr)     # the entropy alone knows no token
    assert not g.isnan().any() and (g[1:] == 0).all()


def test_two_captured_graphs_do_not_share_scratch():
    """Two graphs of the split-row form on different inputs, replayed on two streams at once."""
    from vae_amd import functional as F_
    import vae_amd
    V, k = 131072, 20
    xs = [torch.randn(2, V, generator=gen(i)).to(torch.bfloat16).to(DEV) for i in range(2)]
    toks = [torch.randint(0, V, (2,), generator=gen(9 + i)).to(DEV) for i in range(2)]
    want = [F_.token_log_probs(x, t, top_k=k) for x, t in zip(xs, toks)]
    steps = [vae_amd.graph.capture(lambda x=x, t=t: F_.token_log_probs(x, t, top_k=k)) for x, t in zip(xs, toks)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for s, step in zip(streams, steps):
            with torch.cuda.stream(s):
                step()
    torch.cuda.synchronize()
    for w, step in zip(want, steps):
        for a, b in zip(w, step.outputs):
            assert torch.equal(a, b)


def test_no_rows_and_one_dimensional_logits():
    from vae_amd import functional as F_
    x = torch.randn(0, 30, device=DEV, requires_grad=True)
    lp, h, top, ids = F_.token_log_probs(x, torch.zeros(0, dtype=torch.int64, device=DEV), top_k=2)
    assert lp.shape == (0,) and top.shape == (0, 2) and ids.shape == (0, 2)
    g, = torch.autograd.grad(lp.sum() + h.sum(), x)
    assert g.shape == x.shape
    kl, mean = F_.distill_top_logits(x, torch.zeros(0, 3, device=DEV), torch.zeros(0, 3, dtype=torch.int64, device=DEV))
    assert kl.shape == (0,) and float(mean) == 0.0
    g, = torch.autograd.grad(mean, x)
    assert g.shape == x.shape
    out = F_.nll_elbo(torch.zeros(0, 2, dtype=torch.int64, device=DEV), torch.zeros(0, 2, 5, device=DEV), 'categorical')
    assert out[0].shape == (0,)
    assert bool((F_.nll(torch.zeros(3, 0, dtype=torch.int64, device=DEV), torch.zeros(3, 0, 5, device=DEV),
                        'categorical') == 0).all())
    v = torch.randn(30, device=DEV)
    lp, h, top, ids = F_.token_log_probs(v, torch.tensor(4, device=DEV), top_k=2)
    assert lp.dim() == 0 and top.shape == (2,)
    torch.testing.assert_close(lp, torch.log_softmax(v, 0)[4], rtol=1e-6, atol=4e-6)


def test_many_short_rows_and_offsets_beyond_32_bits():
    """More elements than 2^31: rows whose offsets need 64 bits are read and written where they are."""
    from vae_amd import functional as F_
    N, V = 40000, 65536
    if torch.cuda.get_device_properties(0).total_memory < 40 << 30:
        pytest.skip('needs 11 GB')
    x = torch.empty(N, V, dtype=torch.bfloat16, device=DEV)
    x.normal_(generator=torch.Generator(device=DEV).manual_seed(1))
    tok = torch.full((N,), -1, dtype=torch.int64, device=DEV)
    rows = [0, 32767, 32768, 33000, N - 1]
    tok[rows] = torch.tensor([5, 6, V - 1, 0, 9], device=DEV)
    x.requires_grad_(True)
    _, loss, _, means = F_.nll_elbo(tok[:, None], x[:, None], 'categorical', fuse_backward=True)
    g, = torch.autograd.grad(means[0], x)
    lp, h, top, ids = F_.token_log_probs(x.detach(), tok, top_k=3)
    for r in rows:
        z = x.detach()[r].double().cpu()[None]
        logp, p, hr = ref_rows(z)
        close(lp[r], logp[0, tok[r].cpu()], 1e-6, 4e-6)
        close(h[r], hr[0], 1e-6, 2e-5)
        assert torch.equal(ids[r].cpu(), ref_top(z, 3)[0])
        p[0, tok[r].cpu()] -= 1.0
        check_grad(g[r], p[0] / N, 1.0 / N)
    assert bool((g[1] == 0).all()) and bool((g[N - 2] == 0).all())


@pytest.mark.parametrize('V,dt', [(257, 'bf16'), (300, 'f32')])
def test_more_rows_than_a_launch_has_blocks(V, dt):
    """2^20 rows and some: the workgroups go round again, with the same shared memory."""
    from vae_amd import functional as F_
    N = (1 << 20) + 37
    x = torch.empty(N, V, dtype=TYPES[dt], device=DEV)
    x.normal_(generator=torch.Generator(device=DEV).manual_seed(1))
    if dt == 'f32':
        x = x[:, :V - 1]                       # rows 1200 bytes apart of 299 elements: no short-row form
    V = x.shape[1]
    x = x.detach().requires_grad_(True)
    tok = torch.randint(0, V, (N,), generator=torch.Generator(device=DEV).manual_seed(2), device=DEV)
    lp, h, top, ids = F_.token_log_probs(x, tok, top_k=3)
    g, = torch.autograd.grad([lp, h, top], [x], [torch.ones_like(lp), torch.ones_like(h), torch.ones_like(top)])
    kl, mean = F_.distill_top_logits(x, top.detach(), ids, inv_count=1.0)
    gd, = torch.autograd.grad(mean, x)
    _, _, _, means = F_.nll_elbo(tok[:, None], x[:, None], 'categorical', inv_count=1.0, fuse_backward=True)
    gn, = torch.autograd.grad(means[0], x)
    rows = torch.tensor([0, 1, 5, 36, 37, (1 << 20) - 1, 1 << 20, (1 << 20) + 1, (1 << 20) + 36])
    z = x.detach()[rows.to(DEV)].double().cpu()
    t = tok[rows.to(DEV)].cpu()
    logp, p, hr = ref_rows(z)
    want = ref_top(z, 3)
    at = lambda v: v.detach()[rows.to(DEV)].cpu()
    close(at(lp), logp.gather(1, t[:, None])[:, 0], 1e-6, 4e-6)
    close(at(h), hr, 1e-6, 2e-5)
    assert torch.equal(at(ids), want)
    ref = -4.0 * p - p * (logp + hr[:, None])
    ref[torch.arange(len(rows)), t] += 1.0
    ref.scatter_add_(1, want, torch.ones(len(rows), 3).double())
    check_grad(at(g), ref, 8.0)
    klr, gr = ref_distill(z, logp.gather(1, want), want, 1.0)
    close(at(kl), klr, 1e-6, 2e-5)
    check_grad(at(gd), gr, 2.0)
    q = p.clone()
    q[torch.arange(len(rows)), t] -= 1.0
    check_grad(at(gn), q, 1.0)
    close(means[0], -torch.log_softmax(x.detach().double(), 1).gather(1, tok[:, None]).sum().cpu(), 1e-5, 0.0)


@pytest.mark.parametrize('dt', ['bf16', 'f32'])
@pytest.mark.parametrize('k', [1, 20, 64])
def test_alternatives_of_whole_rows(k, dt):
    """Rows enough that none is split: equal values, masks that leave little, sorted rows, and large values that all sit in
    one thread's share of a long row (more of them than the candidates' list holds)."""
    from vae_amd import functional as F_
    vec = 4 if dt == 'f32' else 8
    N, V = 520, 300000 if dt == 'bf16' else 310000
    x = torch.empty(N, V, dtype=TYPES[dt], device=DEV)
    x.normal_(generator=torch.Generator(device=DEV).manual_seed(k))
    low = float('-inf')
    x[0] = 1.0
    x[1] = low
    x[2] = low
    x[2, [7, 100000, V - 1]] = torch.tensor([1.0, 3.0, 1.0], dtype=x.dtype, device=DEV)
    x[3] = torch.sort(x[3].float())[0].to(x.dtype)
    x[4] = torch.sort(x[4].float(), descending=True)[0].to(x.dtype)
    col = (3 * vec + torch.arange(0, V - 4 * vec, 256 * vec, device=DEV)[:, None]
           + torch.arange(vec, device=DEV)[None]).reshape(-1)
    x[5, col] = (20.0 + torch.arange(col.numel(), device=DEV) * 0.01).to(x.dtype)
    x[6] = torch.randint(-2, 3, (V,), device=DEV).to(x.dtype)
    x[7] = torch.finfo(TYPES[dt]).min
    _, _, top, ids = F_.token_log_probs(x, top_k=k, want_entropy=False)
    for r in list(range(8)) + [100, N - 1]:
        z = x[r].double().cpu()[None]
        want = ref_top(z, k)
        assert torch.equal(ids[r].cpu(), want[0]), r
        close(top[r], ref_rows(z)[0].gather(1, want)[0], 1e-6, 4e-6)


def test_loss_mean_may_be_scaled_in_place():
    """An accumulation loop's loss /= n, as with the other likelihoods."""
    import vae_amd
    z = torch.randn(3, 2, 30, generator=gen(1))
    x = torch.randint(0, 30, (3, 2), generator=gen(2))
    for dt in ('f32', 'bf16'):
        xr = z.to(TYPES[dt]).to(DEV).requires_grad_(True)
        loss = vae_amd.loss_function(xr, x.to(DEV), torch.zeros(3, device=DEV), 'categorical')['loss_mean']
        loss /= 4
        g, = torch.autograd.grad(loss, xr)
        ref = ref_elbo(z.to(TYPES[dt]).double(), x, torch.zeros(3).double(), 1.0)
        close(loss, ref[0].mean() / 4, 2 * HALF[TYPES[dt]] + 1e-6, 1e-5)
        # stored as d(loss_mean), rounded, then scaled by 1/4: exact
        check_grad(g, ref[3] / 12, 0.1)


def test_means_over_many_samples():
    """More samples than one block takes: the means of 10000 x 3 tokens, with KL, additional and mutual-information terms."""
    from vae_amd import functional as F_
    B, T, V = 10000, 3, 20
    z = torch.randn(B, T, V, generator=gen(1))
    x = torch.randint(-1, V, (B, T), generator=gen(2))
    terms = [torch.rand(B, generator=gen(3 + i)) for i in range(3)]
    nll, loss, elbo, means = F_.nll_elbo(x.to(DEV), z.to(DEV), 'categorical', *[t.to(DEV) for t in terms], kl_beta=0.25)
    n = ref_elbo(z.double(), x, torch.zeros(B).double(), 1.0)[0]
    kld, add, mi = [t.double() for t in terms]
    want = torch.stack([(n + add + 0.25 * kld - mi).mean(), (n + kld).mean(), n.mean(), kld.mean(), add.mean(), mi.mean()])
    close(means, want, 2e-6, 1e-6)
    close(loss, n + add + 0.25 * kld - mi, 1e-6, 1e-5)


def test_nan_in_the_loss_raises_the_flag():
    import vae_amd
    vae_amd.nan_flags()
    x = torch.zeros(5, dtype=torch.int64, device=DEV)
    z = torch.randn(5, 12, generator=gen(1)).to(DEV)
    vae_amd.loss_function(z, x, torch.zeros(5, device=DEV), 'categorical')
    assert vae_amd.nan_flags() == 0
    z[3, 4] = float('nan')
    vae_amd.loss_function(z, x, torch.zeros(5, device=DEV), 'categorical')
    assert vae_amd.nan_flags() & 1


def test_second_derivatives_are_refused():
    from vae_amd import functional as F_
    x = torch.randn(3, 9, device=DEV, requires_grad=True)
    tok = torch.tensor([1, 2, 3], device=DEV)
    y = (x * 2).requires_grad_(True)
    lp, _, _, _ = F_.token_log_probs(y, tok)
    g, = torch.autograd.grad(lp.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_expanded_logits():
    """One row shared by several tokens (a broadcast input): its gradient is the sum."""
    from vae_amd import functional as F_
    x = torch.randn(1, 40, generator=gen(1)).to(DEV).requires_grad_(True)
    tok = torch.tensor([3, 5, 5, -1], device=DEV)
    lp, h, _, _ = F_.token_log_probs(x.expand(4, 40), tok)
    g, = torch.autograd.grad(lp.sum(), x)
    p = torch.softmax(x.detach().double().cpu(), 1)
    ref = -3.0 * p
    ref[0, 3] += 1.0
    ref[0, 5] += 2.0
    check_grad(g, ref, 4.0)
    assert bool((h[:3] == h[0]).all()) and float(h[3]) == 0.0


def _slot(i):
    return (i * 2654435761 & 0xffffffff) >> 22


@pytest.mark.parametrize('V,dt', [(5000, 'f32'), (70000, 'bf16')])
@pytest.mark.parametrize('K', [60, 128, 256])
def test_distillation_of_ids_that_come_often(V, K, dt):
    """Many ids many times, many of them in one slot of the table that looks for them, and one id alone."""
    from vae_amd import functional as F_
    one_slot = [i for i in range(V) if _slot(i) == _slot(4321)]
    assert len(one_slot) >= 4
    g = gen(K)
    ids = torch.stack([torch.tensor(one_slot)[torch.randint(0, len(one_slot), (K,), generator=g)],
                       torch.tensor((one_slot * K)[:K]), torch.full((K,), 77), torch.randint(0, V, (K,), generator=g)])
    ids[2, K // 2:] = -1
    z = torch.randn(4, V, generator=g).to(TYPES[dt])
    y = torch.randn(4, K, generator=g)
    kl_ref, grad_ref = ref_distill(z.double(), y.double(), ids, 1.0)
    for fuse in (True, False):
        x = z.to(DEV).requires_grad_(True)
        kl, mean = F_.distill_top_logits(x, y.to(DEV), ids.to(DEV), fuse_backward=fuse)
        close(kl, kl_ref, 1e-6, 2e-5)
        grad, = torch.autograd.grad(mean, x)
        check_grad(grad, grad_ref / 4, 0.25)


@pytest.mark.parametrize('V,dt', [(1050001, 'f32'), (1050001, 'bf16'), (140000, 'bf16')])
@pytest.mark.parametrize('k', [1, 5, 64])
def test_alternatives_over_many_pieces(V, dt, k):
    """More pieces than alternatives, and fewer; equal values, the large ones in one piece."""
    from vae_amd import functional as F_
    z = torch.randn(4, V, generator=gen(k)).to(TYPES[dt])
    z[1] = 0.25
    z[2, V // 2:V // 2 + 90] = 9.0
    z[3] = torch.sort(z[3])[0]
    _, _, top, ids = F_.token_log_probs(z.to(DEV), top_k=k)
    assert torch.equal(ids.cpu(), ref_top(z.double(), k))
    _, _, _, alone = F_.token_log_probs(z[:1].to(DEV), top_k=k)
    assert torch.equal(alone.cpu(), ids[:1].cpu())


@pytest.mark.parametrize('dt', ['f32', 'bf16'])
@pytest.mark.parametrize('V,k', [(200, 64), (512, 7), (512, 8), (512, 48), (512, 49), (513, 49), (1024, 3), (1024, 4),
                                 (1024, 64), (1025, 3), (900, 64), (1790, 49), (1800, 49), (2000, 64), (8192, 48),
                                 (8193, 49)])
def test_alternatives_where_the_kernels_change(V, k, dt):
    from vae_amd import functional as F_
    z = torch.randn(5, V, generator=gen(V + k)).to(TYPES[dt])
    z[1] = -2.0
    z[2, :V - 3] = float('-inf')
    tok = torch.tensor([0, V - 1, V - 2, -1, 5])
    lp, h, top, ids = F_.token_log_probs(z.to(DEV), tok.to(DEV), top_k=k)
    logp, _, hr = ref_rows(z.double())
    live = [0, 1, 2, 4]
    assert torch.equal(ids.cpu()[live], ref_top(z.double(), k)[live])
    assert (ids[3] == -1).all()
    close(lp[live], logp[live, tok[live]], 1e-6, 4e-6)
    close(h[live], hr[live], 1e-6, 2e-5)


def test_many_rows_of_a_wave_each():
    from vae_amd import functional as F_
    N, V = 2100, 8192
    x = torch.randn(N, V, device=DEV, generator=torch.Generator(DEV).manual_seed(1)).to(torch.bfloat16)
    tok = torch.randint(0, V, (N,), generator=gen(2)).to(DEV)
    lp, h, top, ids = F_.token_log_probs(x, tok, top_k=3)
    few = torch.arange(0, N, 37)
    z = x[few.to(DEV)].double().cpu()
    logp, _, hr = ref_rows(z)
    close(lp[few.to(DEV)], logp.gather(1, tok.cpu()[few][:, None])[:, 0], 1e-6, 4e-6)
    close(h[few.to(DEV)], hr, 1e-6, 2e-5)
    assert torch.equal(ids.cpu()[few], ref_top(z, 3))


@pytest.mark.parametrize('B,T', [(1, 70001), (3, 5003), (2, 4096), (700, 9), (1, 1)])
def test_long_sums(B, T):
    """Sums of many rows: in double, rounded once (half a step of fp32), the double sum itself 2^-40 off at most."""
    from vae_amd import functional as F_
    rows = torch.rand(B, T, generator=gen(T)) + 0.5
    got = F_.sample_sums(rows.to(DEV))
    close(got, rows.double().sum(1), 2.0 ** -24 + 2.0 ** -40, 0.0)
    z, x = torch.randn(B, T, 5, generator=gen(B)), torch.randint(0, 5, (B, T), generator=gen(3))
    lp = F_.token_log_probs(z.to(DEV), x.to(DEV), want_entropy=False)[0]
    close(F_.nll(x.to(DEV), z.to(DEV), 'categorical'), -lp.double().cpu().sum(1), 2.0 ** -24 + 2.0 ** -40, 0.0)
    kl, mean = F_.distill_top_logits(z.to(DEV), torch.randn(B, T, 2, generator=gen(4)).to(DEV),
                                     torch.randint(0, 5, (B, T, 2), generator=gen(5)).to(DEV), inv_count=0.25)
    close(mean, 0.25 * kl.double().cpu().sum(), 2.0 ** -24 + 2.0 ** -40, 0.0)
