"""What the categorical-observation entry points refuse, on the host and before any launch: no GPU needed.  The C entry
points return VAE_ERR_ARG for every shape, type or pointer that their kernels could not take."""
import ctypes

import pytest
import torch

from vae_amd import _lib
from vae_amd import functional as F_


def test_python_refusals():
    x = torch.zeros(4, 10)
    tok = torch.zeros(4, dtype=torch.int64)
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        F_.token_log_probs(x, tok)
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        F_.nll(tok, x, 'categorical')
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        F_.distill_top_logits(x, torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.int32))
    with pytest.raises(TypeError):
        F_.token_log_probs(x, tok.float())
    with pytest.raises(TypeError):
        F_.nll(tok.float(), x, 'categorical')
    with pytest.raises(TypeError):
        F_.distill_top_logits(x, torch.zeros(4, 2), torch.zeros(4, 2))
    for k in (-1, 11, 65):
        with pytest.raises(ValueError):
            F_.token_log_probs(torch.zeros(4, 10 if k != 65 else 100), tok, top_k=k)
    with pytest.raises(ValueError):
        F_.token_log_probs(x, tok[:3])
    with pytest.raises(ValueError):
        F_.token_log_probs(torch.zeros(4, 0), tok)
    with pytest.raises(ValueError):
        F_.token_log_probs(torch.zeros(()))
    with pytest.raises(ValueError):
        F_.nll(tok, torch.zeros(4, 3, 10), 'categorical')
    with pytest.raises(ValueError):
        F_.nll(tok, torch.zeros(10), 'categorical')
    ids = torch.zeros(4, 2, dtype=torch.int64)
    with pytest.raises(ValueError):
        F_.distill_top_logits(x, torch.zeros(4, 3), ids)
    with pytest.raises(ValueError):
        F_.distill_top_logits(x, torch.zeros(3, 2), ids[:3])
    with pytest.raises(ValueError):
        F_.distill_top_logits(x, torch.zeros(4, 257), torch.zeros(4, 257, dtype=torch.int64))
    with pytest.raises(ValueError):
        F_.distill_top_logits(x, torch.zeros(4, 0), torch.zeros(4, 0, dtype=torch.int64))
    for tau in (0.0, -1.0, float('nan'), float('inf')):
        with pytest.raises(ValueError):
            F_.distill_top_logits(x, torch.zeros(4, 2), ids, temperature=tau)
    with pytest.raises(ValueError, match='teacher'):
        F_.distill_top_logits(x, torch.zeros(4, 2, requires_grad=True), ids)
    with pytest.raises(TypeError):
        F_.sample_sums(torch.zeros(4, 2, dtype=torch.float64))
    for term in ('kld', 'add', 'mi'):       # the kernel reads one of each for every sample
        with pytest.raises(ValueError, match=term):
            F_.nll_elbo(tok, x, 'categorical', **{term: torch.zeros(3)})


def _call(name, args):
    """The entry point with `args` by position; pointers are host addresses, which nothing may dereference."""
    return getattr(_lib.load(), name)(*args)


P = ctypes.c_void_p(4096)   # never read: every call below is refused, or has no rows


def fwd(**kw):
    a = dict(logits=P, stride=10, tokens=P, tb=8, logp=P, ent=P, stats=P, top=P, ids=P, k=3, scratch=P, N=2, V=10,
             dtype=0)
    a.update(kw)
    return _call('vae_token_logp_fwd', [a[n] for n in ('logits', 'stride', 'tokens', 'tb', 'logp', 'ent', 'stats', 'top',
                                                       'ids', 'k', 'scratch', 'N', 'V', 'dtype')] + [None])


def bwd(**kw):
    a = dict(logits=P, stride=10, tokens=P, tb=8, stats=P, ent=P, glogp=P, per=1, scale=1.0, gent=P, gtop=P, ids=P, k=3,
             out=P, N=2, V=10, dtype=0)
    a.update(kw)
    return _call('vae_token_logp_bwd', [a[n] for n in ('logits', 'stride', 'tokens', 'tb', 'stats', 'ent', 'glogp', 'per',
                                                       'scale', 'gent', 'gtop', 'ids', 'k', 'out', 'N', 'V', 'dtype')]
                 + [None])


def fused(**kw):
    a = dict(logits=P, stride=10, tokens=P, tb=8, T=1, kld=None, add=None, mi=None, beta=1.0, inv=1.0, logp=P, stats=P,
             out=P, nll=P, loss=P, elbo=P, means=P, first=P, others=P, md=0, ws=P, scratch=P, N=2, V=10, dtype=0)
    a.update(kw)
    return _call('vae_token_nll_elbo_fwd',
                 [a[n] for n in ('logits', 'stride', 'tokens', 'tb', 'T', 'kld', 'add', 'mi', 'beta', 'inv', 'logp', 'stats',
                                 'out', 'nll', 'loss', 'elbo', 'means', 'first', 'others', 'md', 'ws', 'scratch', 'N', 'V',
                                 'dtype')]
                 + [None])


def dfwd(**kw):
    a = dict(logits=P, stride=10, y=P, ys=2, yt=0, ids=P, ids_s=2, ib=8, K=2, tau=1.0, t=P, kl=P, mean=None, scale=1.0,
             stats=P, out=P, scratch=P, N=2, V=10, dtype=0)
    a.update(kw)
    return _call('vae_distill_fwd', [a[n] for n in ('logits', 'stride', 'y', 'ys', 'yt', 'ids', 'ids_s', 'ib', 'K', 'tau',
                                                    't', 'kl', 'mean', 'scale', 'stats', 'out', 'scratch', 'N', 'V',
                                                    'dtype')] + [None])


def dbwd(**kw):
    a = dict(logits=P, stride=10, t=P, K=2, tau=1.0, stats=P, gkl=P, gm=P, scale=1.0, out=P, N=2, V=10, dtype=0)
    a.update(kw)
    return _call('vae_distill_bwd', [a[n] for n in ('logits', 'stride', 't', 'K', 'tau', 'stats', 'gkl', 'gm', 'scale',
                                                    'out', 'N', 'V', 'dtype')] + [None])


BAD = [dict(N=-1), dict(V=0), dict(V=(1 << 24) + 1, stride=1 << 25), dict(stride=9), dict(dtype=3), dict(logits=None)]


@pytest.mark.parametrize('f', [fwd, bwd, fused, dfwd, dbwd])
@pytest.mark.parametrize('bad', BAD)
def test_c_entry_points_refuse_bad_shapes(f, bad):
    assert f(**bad) == _lib.VAE_ERR_ARG


@pytest.mark.parametrize('f,bad', [
    (fwd, dict(k=-1)), (fwd, dict(k=65, V=100, stride=100)), (fwd, dict(k=11)), (fwd, dict(tb=2)),
    (fwd, dict(scratch=None, V=65536, stride=65536)), (dfwd, dict(scratch=None, V=65536, stride=65536)),
    (fused, dict(scratch=None, V=65536, stride=65536)), (fwd, dict(tokens=None)), (fwd, dict(top=None)), (fwd, dict(ids=None)),
    (bwd, dict(k=65)), (bwd, dict(k=-1)), (bwd, dict(per=0)), (bwd, dict(stats=None)), (bwd, dict(out=None)),
    (bwd, dict(tb=1)), (bwd, dict(ent=None)), (bwd, dict(gtop=None)), (bwd, dict(ids=None)), (bwd, dict(tokens=None)),
    (fused, dict(tokens=None)), (fused, dict(logp=None)), (fused, dict(stats=None)),
    (fused, dict(tb=0)),
    (dfwd, dict(K=0)), (dfwd, dict(K=257)), (dfwd, dict(tau=0.0)), (dfwd, dict(tau=float('nan'))),
    (dfwd, dict(tau=float('inf'))), (dfwd, dict(t=None)), (dfwd, dict(kl=None)), (dfwd, dict(stats=None)),
    (dfwd, dict(tau=1e-39)), (dbwd, dict(tau=1e-39)),
    (dbwd, dict(K=0)), (dbwd, dict(tau=-1.0)), (dbwd, dict(stats=None)), (dbwd, dict(out=None)), (dbwd, dict(t=None)),
    (dfwd, dict(K=257, ys=300, ids_s=300)), (dfwd, dict(ys=1)), (dfwd, dict(ids_s=1)), (dfwd, dict(ib=2)),
    (dfwd, dict(yt=9)), (dfwd, dict(y=None)), (dfwd, dict(ids=None)),
    (fused, dict(T=-1)), (fused, dict(md=4)), (fused, dict(loss=None)), (fused, dict(elbo=None)),
    (fused, dict(means=None)), (fused, dict(loss=None, elbo=None, nll=None)),
])
def test_c_entry_points_refuse_bad_arguments(f, bad):
    assert f(**bad) == _lib.VAE_ERR_ARG


@pytest.mark.parametrize('f', [fwd, bwd, fused, dfwd, dbwd])
def test_no_rows_is_fine(f):
    assert f(N=0) == _lib.VAE_OK


def test_scratch_sizes():
    lib = _lib.load()
    assert lib.vae_token_scratch_bytes(4096, 131072, 20, 1) == 0          # rows enough: no pieces
    assert lib.vae_token_scratch_bytes(1, 131072, 20, 1) > 0
    for bad in ((0, 100, 0, 0), (1, 0, 0, 0), (1, 100, 65, 0), (1, 100, -1, 0), (1, (1 << 24) + 1, 0, 0)):
        assert lib.vae_token_scratch_bytes(*bad) == 0
    assert lib.vae_distill_teacher_floats(10, 7) == 10 * 22
    assert lib.vae_distill_teacher_floats(10, 0) == lib.vae_distill_teacher_floats(10, 257) == 0


def test_sums_and_scale_refusals():
    assert _call('vae_row_sums', [None, 1.0, P, 2, 3, 0, None]) == _lib.VAE_ERR_ARG
    assert _call('vae_row_sums', [P, 1.0, None, 2, 3, 0, None]) == _lib.VAE_ERR_ARG
    assert _call('vae_row_sums', [P, 1.0, P, -1, 3, 0, None]) == _lib.VAE_ERR_ARG
    assert _call('vae_row_sums', [P, 1.0, P, 2, -3, 0, None]) == _lib.VAE_ERR_ARG
    assert _call('vae_row_sums', [P, 1.0, P, 2, 3, 5, None]) == _lib.VAE_ERR_ARG
    assert _call('vae_row_sums', [None, 1.0, None, 0, 3, 0, None]) == _lib.VAE_OK
    assert _call('vae_grad_scale', [None, P, 4, 0, None]) == _lib.VAE_ERR_ARG
    assert _call('vae_grad_scale', [P, None, 4, 0, None]) == _lib.VAE_ERR_ARG
    assert _call('vae_grad_scale', [P, P, -4, 0, None]) == _lib.VAE_ERR_ARG
    assert _call('vae_grad_scale', [P, P, 4, 7, None]) == _lib.VAE_ERR_ARG
    assert _call('vae_grad_scale', [None, None, 0, 0, None]) == _lib.VAE_OK


def test_loss_backward_refusals():
    b = 'vae_token_nll_elbo_bwd'
    ok = [None, None, None, None, 0, 1.0, 1.0, P, None, 0, None, None, None, 0, 0, None]
    assert _call(b, ok) == _lib.VAE_OK
    for i, v in ((13, -1), (9, -1), (14, 3), (4, 3)):
        assert _call(b, ok[:i] + [v] + ok[i + 1:]) == _lib.VAE_ERR_ARG
    assert _call(b, [P] + ok[1:8] + [P] + ok[9:]) == _lib.VAE_ERR_ARG              # a stored gradient and per-sample ones
