"""Which steps the categorical per-step loss refuses, before any launch: no GPU needed."""
import pytest
import torch

from vae_amd import functional as F_


@pytest.mark.parametrize('sizes', [(3, 2, 4), (3, 4, 2), (2, 3)])
def test_steps_of_different_batches_are_refused(sizes):
    """Also where they hold T B entries together: the averages over the steps would mix samples."""
    xs = [torch.zeros(b, 2, dtype=torch.int64) for b in sizes]
    recons = [torch.zeros(b, 2, 10) for b in sizes]
    with pytest.raises(ValueError, match='same shapes'):
        F_.nll_steps_elbo(xs, recons, 'categorical')


def test_steps_of_different_types_or_vocabularies_are_refused():
    x = torch.zeros(3, dtype=torch.int64)
    for other in (torch.zeros(3, 10, dtype=torch.bfloat16), torch.zeros(3, 11), torch.zeros(3, 2, 10)):
        with pytest.raises(ValueError, match='same shapes'):
            F_.nll_steps_elbo([x, x], [torch.zeros(3, 10), other], 'categorical')
    with pytest.raises(ValueError, match='same shapes'):
        F_.nll_steps_elbo([x, x.repeat(2)], [torch.zeros(3, 10)] * 2, 'categorical')


def test_steps_of_one_size_in_another_shape_pass():
    """[B] and [B, 1] tokens are the same: they get as far as the device check."""
    x, r = torch.zeros(3, dtype=torch.int32), torch.zeros(3, 10)
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        F_.nll_steps_elbo([x, x[:, None], x.long()], [r, r[:, None], r], 'categorical')


def test_many_steps_of_different_batches_are_refused():
    """Beyond the steps of one launch, without a host model."""
    from vae_amd import vrnn

    class Latent:
        def kl(self, dist_a, prior=None):
            return dist_a

    sizes = [3, 2, 4] * 50
    xs, recons = [torch.zeros(b, dtype=torch.int64) for b in sizes], [torch.zeros(b, 10) for b in sizes]
    params = [{'posterior': torch.zeros(b), 'prior': None} for b in sizes]
    config = {'nll_type': 'categorical', 'kl_beta': 1.0, 'use_prior_kl': False}
    with pytest.raises(ValueError, match='same shapes'):
        vrnn.loss_function(Latent(), config, recons, xs, params)
    same = [torch.zeros(3, dtype=torch.int64)] * 150, [torch.zeros(3, 10)] * 150, params[:1] * 150
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        vrnn.loss_function(Latent(), config, same[1], same[0], same[2])


def test_types_of_the_terms():
    """The C entry points refuse a type that they do not know, where there are terms; without any it is not looked at."""
    import ctypes
    from vae_amd import _lib
    lib, P = _lib.load(), ctypes.c_void_p(4096)   # never read: every call is refused, or has no samples

    def fwd(kld, terms_dtype, B):
        return lib.vae_token_nll_elbo_terms_fwd(P, 10, P, 8, 1, kld, None, None, terms_dtype, 1.0, 1.0, P, P, P, P, P, P, P, P,
                                                P, 0, P, P, B, 10, 0, None)

    def bwd(gkld, terms_dtype, B):
        return lib.vae_token_nll_elbo_terms_bwd(None, None, None, None, 0, 1.0, 1.0, P, None, 0, gkld, None, None, terms_dtype,
                                                B, 0, None)

    for f in (fwd, bwd):
        assert f(P, 3, 2) == f(P, -1, 2) == _lib.VAE_ERR_ARG
        assert f(P, 3, 0) == _lib.VAE_ERR_ARG
        assert f(None, 3, 0) == f(P, 2, 0) == _lib.VAE_OK


def test_capture_number_needs_a_place():
    from vae_amd import _lib
    assert _lib.load().vae_capture_id(None, None) == _lib.VAE_ERR_ARG


def test_scratch_is_what_the_library_asks_for():
    """The binding knows no limits of its own: rows that the kernels would cut get the bytes that they ask for."""
    from vae_amd import _lib
    lib = _lib.load()
    cut = 0
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        for N in (1, 2, 64, 255, 256, 257, 4096):
            for V in (1, 1000, 32767, 32768, 65535, 65536, 65543, 131071, 131072, 1 << 20):
                for k in (0, 5, 64):
                    want = lib.vae_token_scratch_bytes(N, V, min(k, V), _lib.DTYPE_CODES[dtype])
                    got = F_._token_scratch(torch.empty((N, V), dtype=dtype, device='meta'), min(k, V), 'meta')
                    assert (0 if got is None else got.numel()) == want
                    cut += want > 0
    assert cut > 50
    assert F_._teacher_floats(10, 7) == lib.vae_distill_teacher_floats(10, 7)
