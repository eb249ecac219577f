"""Categorical observations where they can go wrong: gradients inside a larger buffer, small temperatures, logits far apart,
terms of another type or shape.  Against float64 on the CPU.

Gradients are checked element by element.  p_j = 2^d / s: d = (x - m) c takes two roundings, at most |d| 2^-23 off in the
exponent, 64 2^-23 ln2 = 5.3e-6 of p where |d| <= 64; v_exp_f32 and the sum add less than 2.5e-6 (V <= 2^18 terms in 256 or
more partial sums).  So p is within 8e-6 of itself and the result is rounded once: eps / 2.  Only where an entry is added to
it (the token's, the teacher's) do two terms cancel: there 8e-6 of the upstream factor, absolutely."""
import pytest
import torch

from vae_amd import _lib

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def check_elements(g, ref, entries, scale, more=0.0, floor=0.0):
    """`entries`: truth values, where a second term was added; `scale`: the upstream factor; `more`: another rounding;
    `floor`: what need not be there."""
    tol = (torch.finfo(g.dtype).eps / 2 + 8e-6 + more) * ref.abs() + scale * (8e-6 * entries + floor)
    if g.dtype == torch.float16:
        tol = tol + 2.0 ** -25                     # half a step of its subnormals
    off = (g.detach().double().cpu() - ref).abs()
    worst = (off / tol.clamp(min=1e-300)).max()
    assert bool((off <= tol).all()), 'up to %g times the tolerance' % worst


# ---------------------------------------------------------------------------------------------------------------------
# memory around a gradient
# ---------------------------------------------------------------------------------------------------------------------
GUARD = 150000          # elements: more than the longest piece a workgroup stores


class Guarded:
    """[N, V] inside a buffer of sevens, `off` elements behind a 16-byte boundary."""

    def __init__(self, N, V, dtype, off):
        self.all = torch.full((N * V + 2 * GUARD + 8,), 7.0, dtype=dtype, device=DEV)
        self.lo, self.hi = GUARD + off, GUARD + off + N * V
        self.rows = self.all[self.lo:self.hi].view(N, V)

    def check(self):
        assert bool((self.all[:self.lo] == 7).all()) and bool((self.all[self.hi:] == 7).all())


@pytest.mark.parametrize('dt', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('V', [3, 8, 9, 300, 1500, 5000, 20000, 50021, 70001, 140001])
@pytest.mark.parametrize('off', [0, 1])
def test_nothing_is_written_beside_a_gradient(V, dt, off):
    """Padded rows, the last one among them, in every gradient kernel: the fill of a row or a piece that is shorter than its
    workgroup stays inside it, and the rows in front of it keep their values."""
    N, dtype = 4, TYPES[dt]
    code = _lib.DTYPE_CODES[dtype]
    dev = torch.device(DEV)
    x = (torch.randn(N, V, generator=gen(V)) * 2).to(dtype)
    z = x.double()
    xd = x.to(DEV)
    new = lambda *s: torch.empty(s, dtype=torch.float32, device=DEV)
    p_ = _lib.ptr
    tok = torch.tensor([V // 2, -1, V - 1, -1])
    td = tok.to(DEV)
    live = tok >= 0
    logp = torch.log_softmax(z, -1)
    p = logp.exp() * live[:, None]
    at = torch.zeros(N, V, dtype=torch.bool)
    at[torch.arange(N), tok.clamp(min=0)] = live
    scratch = torch.empty(_lib.load().vae_token_scratch_bytes(N, V, 0, code) + 8, dtype=torch.uint8, device=DEV)

    lp, stats = new(N), new(N, 2)
    _lib.launch(dev, 'vae_token_logp_fwd', p_(xd), V, p_(td), 8, p_(lp), None, p_(stats), None, None, 0, p_(scratch), N, V,
                code)
    g = Guarded(N, V, dtype, off)
    w = torch.tensor([0.5, 3.0, -2.0, 4.0])
    wd = w.to(DEV)
    _lib.launch(dev, 'vae_token_logp_bwd', p_(xd), V, p_(td), 8, p_(stats), None, p_(wd), 1, 1.0, None, None, None, 0,
                p_(g.rows), N, V, code)
    g.check()
    check_elements(g.rows, w.double()[:, None] * (at.double() - p), at, 2.0)

    nll, buf = torch.empty(N, dtype=dtype, device=DEV), new(3 * N)
    g = Guarded(N, V, dtype, off)
    _lib.launch(dev, 'vae_token_nll_elbo_fwd', p_(xd), V, p_(td), 8, 1, None, None, None, 0.0, 0.25, buf.data_ptr(),
                buf.data_ptr() + 4 * N, p_(g.rows), p_(nll), None, None, None, None, None, 0, None, p_(scratch), N, V, code)
    g.check()
    check_elements(g.rows, 0.25 * (p - at.double()), at, 0.25)

    K, tau = 3, 1.5
    y = torch.randn(N, K, generator=gen(1))
    ids = torch.randint(0, V, (N, K), generator=gen(2))
    ids[1] = ids[3] = -1
    yd, idd = y.to(DEV), ids.to(DEV)
    teacher, kl = new(_lib.load().vae_distill_teacher_floats(N, K)), new(N)
    q = torch.softmax(y.double() / tau, -1) * live[:, None]
    ref = torch.softmax(z / tau, -1) * live[:, None]
    ref.scatter_add_(1, ids.clamp(min=0), -q)
    at = torch.zeros(N, V, dtype=torch.bool)
    at.scatter_(1, ids.clamp(min=0), True)
    g = Guarded(N, V, dtype, off)
    _lib.launch(dev, 'vae_distill_fwd', p_(xd), V, p_(yd), K, 0, p_(idd), K, 8, K, tau, p_(teacher), p_(kl), None, 0.5,
                p_(stats), p_(g.rows), p_(scratch), N, V, code)
    g.check()
    check_elements(g.rows, 0.5 / tau * ref, at, 0.5 / tau)
    g = Guarded(N, V, dtype, off)
    _lib.launch(dev, 'vae_distill_bwd', p_(xd), V, p_(teacher), K, tau, p_(stats), p_(wd), None, 0.0, p_(g.rows), N, V, code)
    g.check()
    check_elements(g.rows, w.double()[:, None] / tau * ref, at, 2.0 / tau)


# ---------------------------------------------------------------------------------------------------------------------
# small temperatures
# ---------------------------------------------------------------------------------------------------------------------
def ref_distill(z, y, ids, tau):
    """kl [N], d kl / d z and where the teacher's entries are; float64, every id there"""
    logp, q = torch.log_softmax(z / tau, -1), torch.softmax(y / tau, -1)
    logq = torch.log_softmax(y / tau, -1)
    kl = torch.where(q > 0, q * (logq - logp.gather(1, ids)), torch.zeros_like(q)).sum(1)
    grad = logp.exp() / tau
    grad.scatter_add_(1, ids, -q / tau)
    at = torch.zeros(z.shape, dtype=torch.bool)
    at.scatter_(1, ids, True)
    return kl, grad, at


@pytest.mark.parametrize('dt', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('N,V', [(3, 90), (3, 9000), (2, 70001), (300, 2500)])
@pytest.mark.parametrize('tau,shift', [(1e-4, 0.0), (1e-9, 0.0), (1e-30, 0.0), (1e-4, 6e5), (1e-9, -6e4), (3e-7, 11.3)])
def test_small_temperatures(N, V, dt, tau, shift):
    """x / tau beyond what float32 holds to a unit: one pass, two passes and evaluation agree with float64.  c = log2(e) / tau
    is rounded too, a third step of the exponent: 60 2^-24 ln2 = 2.5e-6 of p more where |d| <= 60; a probability below 2^-60
    of the row's largest need not be there.  The KL's largest term is one such q times a number of five roundings."""
    from vae_amd import functional as F_
    shift = max(min(shift, 6e4), -6e4) if dt == 'f16' else shift
    z = (torch.randn(N, V, generator=gen(V)) * 3 + shift).to(TYPES[dt])
    K = 4
    ids = torch.stack([torch.randperm(V, generator=gen(i))[:K] for i in range(N)])
    y = torch.randn(N, K, generator=gen(2)) * 3 + shift
    kl_r, grad_r, at = ref_distill(z.double(), y.double(), ids, tau)
    w = torch.rand(N, generator=gen(8)) + 0.5

    def near(kl):
        torch.testing.assert_close(kl.detach().double().cpu(), kl_r, rtol=1.2e-5, atol=2e-5)

    with torch.no_grad():
        near(F_.distill_top_logits(z.to(DEV), y.to(DEV), ids.to(DEV), temperature=tau)[0])
    for fuse in (True, False):
        x = z.to(DEV).requires_grad_(True)
        kl, mean = F_.distill_top_logits(x, y.to(DEV), ids.to(DEV), temperature=tau, fuse_backward=fuse)
        near(kl)
        # upstream factors of tau: gradients around 1.  The stored one is rounded, multiplied and rounded again
        g, = torch.autograd.grad(mean, x, torch.tensor(tau, device=DEV), retain_graph=True)
        more = 3e-6 + (torch.finfo(g.dtype).eps / 2 if fuse else 0.0)
        check_elements(g, grad_r * tau / N, at, 1.5 / N, more, 2.0 ** -60)
        g, = torch.autograd.grad(kl, x, (w * tau).to(DEV))
        check_elements(g, grad_r * (w.double() * tau)[:, None], at, 1.5, 3e-6, 2.0 ** -60)


# ---------------------------------------------------------------------------------------------------------------------
# the ELBO's terms
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('fuse', [True, False])
@pytest.mark.parametrize('B,shape', [(4, (4, 1)), (1, ()), (6, (2, 3))])
def test_terms_of_another_shape(B, shape, fuse):
    """A value for each sample, in whatever shape: forward, and each gradient in its term's shape."""
    import vae_amd
    z, x = torch.randn(B, 3, 40, generator=gen(1)), torch.randint(0, 40, (B, 3), generator=gen(2))
    leaves = [torch.rand(shape, generator=gen(3 + i)).to(DEV).requires_grad_(True) for i in range(3)]
    xr = z.to(DEV).requires_grad_(True)
    out = vae_amd.loss_function(xr, x.to(DEV), leaves[0], 'categorical', kl_beta=0.5, mut_info=leaves[2],
                                extra_loss_terms={'more': leaves[1]}, fuse_backward=fuse)
    nll = -torch.log_softmax(z.double(), -1).gather(2, x[..., None])[..., 0].sum(1)
    k, a, m = (t.detach().double().cpu().reshape(-1) for t in leaves)
    torch.testing.assert_close(out['loss'].double().cpu(), nll + a + 0.5 * k - m, rtol=1e-6, atol=1e-5)
    gs = torch.autograd.grad(out['loss_mean'], [xr] + leaves)
    for g, want, t in zip(gs[1:], (0.5 / B, 1.0 / B, -1.0 / B), leaves):
        assert g.shape == t.shape
        torch.testing.assert_close(g, torch.full_like(g, want), rtol=2.0 ** -22, atol=0.0)
    at = torch.zeros(z.shape, dtype=torch.bool).scatter_(2, x[..., None], True)
    check_elements(gs[0], (torch.softmax(z.double(), -1) - at.double()) / B, at, 1.0 / B)


@pytest.mark.parametrize('dt', ['bf16', 'f16'])
@pytest.mark.parametrize('types', [('float32', 'float32', 'float32'), ('float32', 'float64', 'bfloat16'),
                                   ('float16', 'bfloat16', 'float32'), ('bfloat16', 'bfloat16', 'bfloat16')])
@pytest.mark.parametrize('fuse', [True, False])
def test_terms_of_another_type(dt, types, fuse):
    """16-bit logits beside terms of other types: the terms are added as they are, every output is rounded once (half a step
    beside a few of float32), as in the multi-sample form of the same loss; gradients in the terms' own types."""
    from vae_amd import functional as F_
    B, T, V = 7, 5, 300
    z = torch.randn(B, T, V, generator=gen(1)).to(TYPES[dt])
    x = torch.randint(0, V, (B, T), generator=gen(2))
    terms = [(torch.rand(B, generator=gen(3 + i)) * 30).to(getattr(torch, t)) for i, t in enumerate(types)]
    kld, add, mi = (t.double() for t in terms)
    leaves = [t.to(DEV).requires_grad_(True) for t in terms]
    xr = z.to(DEV).requires_grad_(True)
    out = F_.nll_elbo(x.to(DEV), xr, 'categorical', *leaves, kl_beta=0.5, fuse_backward=fuse)
    multi = F_.nll_multi_elbo(x.to(DEV), [z.to(DEV)], 'categorical', *[t.detach() for t in leaves], kl_beta=0.5)
    nll = -torch.log_softmax(z.double(), -1).gather(2, x[..., None])[..., 0].sum(1)
    half = torch.finfo(TYPES[dt]).eps / 2
    loss = nll + add + 0.5 * kld - mi
    means = torch.stack([loss.mean(), (nll + kld).mean(), nll.mean(), kld.mean(), add.mean(), mi.mean()])
    for o in (out, multi):
        for got, want in zip(o, (nll, loss, nll + kld)):
            assert got.dtype == TYPES[dt]
            torch.testing.assert_close(got.double().cpu(), want, rtol=half + 1e-6, atol=1e-5)
        torch.testing.assert_close(o[3].double().cpu(), means, rtol=1e-6, atol=1e-5)
    gs = torch.autograd.grad(out[3][0], leaves)
    for g, want, t in zip(gs, (0.5 / B, 1.0 / B, -1.0 / B), terms):
        assert g.dtype == t.dtype
        torch.testing.assert_close(g.double().cpu(), torch.full((B,), want, dtype=torch.float64),
                                   rtol=torch.finfo(t.dtype).eps / 2 + 2.0 ** -22, atol=0.0)


# ---------------------------------------------------------------------------------------------------------------------
# gradients, element by element
# ---------------------------------------------------------------------------------------------------------------------
ROWS = [(5, 250), (7, 1024), (6, 5000), (3, 40000), (3, 65536), (2, 70001), (80, 98304), (66, 131072), (2, 131072), (1, 140001)]


@pytest.mark.parametrize('dt', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('N,V', ROWS)
@pytest.mark.parametrize('fuse', [True, False])
def test_probabilities_far_below_the_largest(N, V, dt, fuse):
    """Logits evenly spread over 70 units: probabilities down to 2^-101 of the largest, each of which has its bits in the
    likelihood's and the distillation's gradient (d up to 101: 4e-6 more than where it ends at 64)."""
    from vae_amd import functional as F_
    z = (-70.0 * torch.rand(N, V, generator=gen(V))).to(TYPES[dt])
    tok = torch.randint(0, V, (N, 1), generator=gen(1))
    x = z.to(DEV).requires_grad_(True)
    g, = torch.autograd.grad(F_.nll_elbo(tok.to(DEV), x[:, None], 'categorical', fuse_backward=fuse)[3][0], x)
    p = torch.softmax(z.double(), -1)
    at = torch.zeros(N, V, dtype=torch.bool).scatter_(1, tok, True)
    check_elements(g, (p - at.double()) / N, at, 1.0 / N, 4e-6)
    ids = torch.randint(0, V, (N, 3), generator=gen(2))
    y = torch.randn(N, 3, generator=gen(3))
    _, grad, at = ref_distill(z.double(), y.double(), ids, 1.0)
    g, = torch.autograd.grad(F_.distill_top_logits(x, y.to(DEV), ids.to(DEV), fuse_backward=fuse)[1], x)
    check_elements(g, grad / N, at, 1.0 / N, 4e-6)


@pytest.mark.parametrize('dt', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('N,V', [(5, 250), (7, 1024), (6, 5001), (3, 40000), (2, 131072)])
@pytest.mark.parametrize('spread', [9.0, 60.0])
def test_log_prob_entropy_and_alternatives_gradients(N, V, dt, spread):
    """g_j = -p_j (a + b (ln p_j + H)) and the entries.  Its error is p_j times that of the bracket: 1.2e-5 of each product in
    it (p's own error included), and b times the entropy's 2e-5."""
    from vae_amd import functional as F_
    z = (-spread * torch.rand(N, V, generator=gen(V))).to(TYPES[dt])
    tok = torch.randint(0, V, (N,), generator=gen(1))
    a, b, c = (torch.randn(s, generator=gen(2 + i)) for i, s in enumerate([(N,), (N,), (N, 5)]))
    x = z.to(DEV).requires_grad_(True)
    lp, h, top, ids = F_.token_log_probs(x, tok.to(DEV), top_k=5)
    g, = torch.autograd.grad([lp, h, top], x, [t.to(DEV) for t in (a, b, c)])
    logp = torch.log_softmax(z.double(), -1)
    p = logp.exp()
    H = -(p * logp).sum(-1, keepdim=True)
    A, b = (a.double() + c.double().sum(1))[:, None], b.double()[:, None]
    ref = -p * (A + b * (logp + H))
    ref[torch.arange(N), tok] += a.double()
    ref.scatter_add_(1, ids.cpu(), c.double())
    at = torch.zeros(N, V, dtype=torch.bool).scatter_(1, ids.cpu(), True).scatter_(1, tok[:, None], True)
    entries = a.abs().double()[:, None] + c.abs().double().sum(1, keepdim=True)
    tol = torch.finfo(g.dtype).eps / 2 * ref.abs() + 8e-6 * at * entries
    tol = tol + p * (1.2e-5 * (entries + b.abs() * (logp.abs() + H)) + 2e-5 * b.abs())
    if dt == 'f16':
        tol = tol + 2.0 ** -25
    off = (g.double().cpu() - ref).abs()
    assert bool((off <= tol).all()), 'up to %g times the tolerance' % (off / tol.clamp(min=1e-300)).max()


@pytest.mark.parametrize('kind', ['nll', 'distill'])
@pytest.mark.parametrize('dt', ['f32', 'bf16'])
def test_forward_and_backward_in_graphs_of_their_own(kind, dt):
    """A backward graph replayed more often than its forward graph, upstream gradient 2: the same each time, also after the
    logits have changed and the forward graph has been replayed."""
    from vae_amd import functional as F_
    N, V = 12, 3000
    x = (torch.randn(N, V, generator=gen(3)) * 2).to(TYPES[dt])
    tok = torch.randint(0, V, (N, 1), generator=gen(4))
    y, ids = torch.randn(N, 5, generator=gen(5)), torch.stack([torch.randperm(V, generator=gen(i))[:5] for i in range(N)])
    td, yd, idd = tok.to(DEV), y.to(DEV), ids.to(DEV)

    def loss(x):
        if kind == 'nll':
            return F_.token_nll_elbo(td, x[:, None], fuse_backward=True)[3][0]
        return F_.distill_top_logits(x, yd, idd)[1]

    def check(g, z):
        if kind == 'nll':
            at = torch.zeros(N, V, dtype=torch.bool).scatter_(1, tok, True)
            check_elements(g, (torch.softmax(z, -1) - at.double()) * 2.0 / N, at, 2.0 / N)
        else:
            _, ref, at = ref_distill(z, y.double(), ids, 1.0)
            check_elements(g, ref * 2.0 / N, at, 2.0 / N)

    two = torch.full((), 2.0, device=DEV)
    static = x.to(DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            leaf = static.detach().requires_grad_(True)
            torch.autograd.grad(loss(leaf), leaf, two)
    torch.cuda.synchronize()
    leaf = static.detach().requires_grad_(True)
    forward, backward = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(forward, stream=s):
        value = loss(leaf)
    with torch.cuda.graph(backward, stream=s):
        g, = torch.autograd.grad(value, leaf, two)
    for turn in range(3):
        z = x.flip(1) if turn == 1 else x
        static.copy_(z)
        forward.replay()
        for _ in range(3):
            backward.replay()
            torch.cuda.synchronize()
            check(g, z.double())
            g.zero_()
            torch.cuda.synchronize()


def test_forward_and_backward_in_one_graph_keep_the_stored_gradient():
    """... and replays of one graph that holds both are right with an upstream gradient of 2, too."""
    import vae_amd
    from vae_amd import functional as F_
    N, V = 9, 2000
    x = torch.randn(N, V, generator=gen(3))
    tok = torch.randint(0, V, (N, 1), generator=gen(4))
    static, td, two = x.to(DEV), tok.to(DEV), torch.full((), 2.0, device=DEV)

    def step():
        leaf = static.detach().requires_grad_(True)
        return torch.autograd.grad(F_.token_nll_elbo(td, leaf[:, None], fuse_backward=True)[3][0], leaf, two)[0]

    replay = vae_amd.graph.capture(step)
    at = torch.zeros(N, V, dtype=torch.bool).scatter_(1, tok, True)
    for turn in range(4):
        z = x.flip(1) if turn % 2 else x
        static.copy_(z)
        g = replay()
        torch.cuda.synchronize()
        check_elements(g, (torch.softmax(z.double(), -1) - at.double()) * 2.0 / N, at, 2.0 / N, 2.0 ** -24)


@pytest.mark.parametrize('dt,V', [('f32', 50), ('bf16', 9000), ('f16', 9000), ('bf16', 70000), ('f32', 70001)])
@pytest.mark.parametrize('fuse', [True, False])
def test_a_teacher_without_a_distribution_makes_its_row_nan(dt, V, fuse):
    """NaN or +inf among the teacher's logits: kl and the whole row's gradient, (sum q) p - q, are NaN; the other rows are
    what they are without it."""
    from vae_amd import functional as F_
    N = 5
    z = torch.randn(N, V, generator=gen(V)).to(TYPES[dt])
    ids = torch.stack([torch.randperm(V, generator=gen(i))[:4] for i in range(N)])
    y = torch.randn(N, 4, generator=gen(1))
    kl_r, grad_r, at = ref_distill(z.double(), y.double(), ids, 1.0)
    y[1, 2] = float('nan')
    y[3, 0] = float('inf')
    bad, fine = [1, 3], [0, 2, 4]
    x = z.to(DEV).requires_grad_(True)
    kl, mean = F_.distill_top_logits(x, y.to(DEV), ids.to(DEV), fuse_backward=fuse)
    assert bool(kl[bad].isnan().all()) and bool(mean.isnan())
    torch.testing.assert_close(kl[fine].detach().double().cpu(), kl_r[fine], rtol=1e-6, atol=2e-5)
    for out, up, scale in ((mean, torch.ones(()), 1.0 / N), (kl, torch.ones(N), 1.0)):
        g, = torch.autograd.grad(out, x, up.to(DEV), retain_graph=True)
        assert bool(g[bad].isnan().all())
        check_elements(g[fine], grad_r[fine] * scale, at[fine], scale)
