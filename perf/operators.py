"""The categorical-observation operators: log probabilities of given tokens (with entropy and the top alternatives), the
categorical likelihood inside the ELBO loss, and distillation from a teacher's top logits.

`listed()` / `draw()` give cases, `prepare()` a case's inputs on the GPU, `run()` one pass: through this package's entry
points when `own` is true, else the plain form (elementary torch operations in float32, rounded once at the end).
`exact()` is the same from the definitions in float64.

Conventions of the operators: logits [..., V]; a negative token marks a padded row (log prob 0, entropy 0, alternatives
-inf / -1, gradient 0); logits of -inf are masked out; alternatives are ordered by value, ties by the lower index.
"""
import math

import torch

own = False

DEV = 'cuda'
TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
SIZE = {'f32': 4, 'bf16': 2, 'f16': 2}


def listed():
    return [
        # one new token of one sequence: its alternatives, nothing to hide a launch behind
        dict(name='serve_one', op='score', B=1, T=1, V=32768, k=5, entropy=True, dtype='bf16', pad=0.0, masked=0.0),
        # a serving batch of new tokens over a large vocabulary, part of it masked by a grammar
        dict(name='serve_batch', op='score', B=64, T=1, V=131072, k=20, entropy=True, dtype='bf16', pad=0.0, masked=0.4),
        # a handful of sequences, logits left in float32 by the head, a vocabulary that breaks alignment
        dict(name='serve_odd_f32', op='score', B=7, T=1, V=50021, k=8, entropy=False, dtype='f32', pad=0.0, masked=0.0),
        # scoring ragged prompts: every position's token and a few alternatives, rows behind a sequence's end padded
        dict(name='score_ragged', op='score', B=16, T=128, V=50021, k=4, entropy=True, dtype='f16', pad=0.3, masked=0.0),
        # policy-gradient step with an entropy bonus, small: latency of forward plus backward
        dict(name='policy_small', op='policy', B=96, T=1, V=1000, k=0, entropy=True, dtype='f32', pad=0.0, masked=0.0),
        # the same at training size
        dict(name='policy_train', op='policy', B=32, T=128, V=32768, k=0, entropy=True, dtype='bf16', pad=0.1, masked=0.0),
        # one recurrent step's categorical likelihood: 64 samples, 1024 categories
        dict(name='elbo_step', op='elbo', B=64, T=1, V=1024, dtype='f32', pad=0.0),
        # 28 x 28 pixels of 256 levels each: short rows, many of them
        dict(name='elbo_pixels', op='elbo', B=256, T=784, V=256, dtype='bf16', pad=0.0),
        # a text decoder's loss: long rows, ragged sequences
        dict(name='elbo_text', op='elbo', B=16, T=509, V=65536, dtype='bf16', pad=0.1),
        # distillation, small: latency
        dict(name='distill_small', op='distill', B=128, V=4097, K=16, tau=1.0, how='mean', dtype='f32', pad=0.0),
        # per-row weights (a loss mask of the user's own): the gradient arrives row by row; odd sizes
        dict(name='distill_rows', op='distill', B=1021, V=50021, K=33, tau=2.0, how='rows', dtype='f16', pad=0.2),
        # a full distillation step: mean loss and its gradient
        dict(name='distill_train', op='distill', B=4096, V=131072, K=64, tau=2.0, how='mean', dtype='bf16', pad=0.0),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(['score', 'score', 'policy', 'elbo', 'distill'])
    dtype = rng.choice(['bf16', 'bf16', 'f16', 'f32'])
    V = _spread(rng, 40, 150000)
    rows = _spread(rng, 1, max(1, min(200000, (1 << 28) // V)))
    T = rng.choice([1, _spread(rng, 1, rows)])
    B = max(1, rows // T)
    pad = rng.choice([0.0, round(rng.uniform(0.05, 0.5), 2)])
    if op == 'score':
        return dict(op=op, B=B, T=T, V=V, k=rng.choice([0, rng.randint(1, min(V, 24))]), entropy=rng.random() < 0.7,
                    dtype=dtype, pad=pad, masked=rng.choice([0.0, round(rng.uniform(0.1, 0.9), 2)]))
    if op == 'policy':
        return dict(op=op, B=B, T=T, V=V, k=0, entropy=rng.random() < 0.7, dtype=dtype, pad=pad,
                    masked=rng.choice([0.0, round(rng.uniform(0.1, 0.9), 2)]))
    if op == 'elbo':
        if dtype == 'f16':
            T = min(T, 1000)                       # a sample's summed nll has to fit the type it is returned in
        return dict(op=op, B=B, T=T, V=V, dtype=dtype, pad=pad)
    return dict(op=op, B=B * T, V=V, K=rng.randint(1, min(V, 128)), tau=round(rng.uniform(0.7, 4.0), 2),
                how=rng.choice(['mean', 'rows', 'eval']), dtype=dtype, pad=pad)


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _live_rows(case):
    """How many positions of each sequence are real: lengths between (1 - 2 pad) T and T, at least one."""
    B, T = case['B'], case.get('T', 1)
    if T == 1:
        return None
    low = max(1, int(T * (1.0 - 2.0 * case['pad'])))
    return [low + (b * 7919) % (T - low + 1) for b in range(B)]


def _padding(case):
    """[rows] bool on the GPU: True where a row is padding."""
    B, T = case['B'], case.get('T', 1)
    lengths = _live_rows(case)
    if lengths is None:
        return torch.arange(B, device=DEV) >= B - int(B * case['pad'])
    if case['pad'] == 0.0:
        return torch.zeros(B * T, dtype=torch.bool, device=DEV)
    return (torch.arange(T, device=DEV)[None] >= torch.tensor(lengths, device=DEV)[:, None]).reshape(-1)


def _live_count(case):
    B, T = case['B'], case.get('T', 1)
    lengths = _live_rows(case)
    if lengths is None:
        return B - int(B * case['pad'])
    return B * T if case['pad'] == 0.0 else sum(lengths)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = TYPES[case['dtype']]
    B, T, V = case['B'], case.get('T', 1), case['V']
    N = B * T
    # a head's logits: a wide bulk, and the token that comes next well above it most of the time
    x = torch.randn(N, V, generator=g, device=DEV, dtype=torch.float32).mul_(2.5)
    padding = _padding(case)
    state = dict(case=case)
    if case['op'] == 'distill':
        K = case['K']
        # K different ids a row, and logits sorted as a top-K comes
        first = torch.randint(0, V, (N, 1), generator=g, device=DEV)
        step = torch.randint(1, max(V // K, 1) + 1, (N, 1), generator=g, device=DEV)
        ids = (first + step * torch.arange(K, device=DEV)[None]) % V
        teacher = torch.randn(N, K, generator=g, device=DEV).mul_(3.0).sort(-1, descending=True)[0] + 8.0
        x.scatter_add_(1, ids, 0.7 * teacher)       # the student has learned some of it
        if case['pad'] > 0.0:
            ids = torch.where(padding[:, None], torch.full_like(ids, -1), ids)
        state.update(ids=ids.to(torch.int32), teacher=teacher.to(dt))
        if case['how'] == 'rows':
            state['weights'] = torch.rand(N, generator=g, device=DEV)
        state['logits'] = x.to(dt).requires_grad_(case['how'] != 'eval')
        return state
    tokens = torch.randint(0, V, (N,), generator=g, device=DEV)
    x.scatter_add_(1, tokens[:, None], torch.rand(N, 1, generator=g, device=DEV) * 10.0)
    if case.get('masked', 0.0) > 0.0:
        hide = torch.rand(V, generator=g, device=DEV)[None].expand(N, V) < case['masked']
        hide = hide.scatter(1, tokens[:, None], False)
        x.masked_fill_(hide, float('-inf'))
    tokens = torch.where(padding, torch.full_like(tokens, -100), tokens)
    if case['op'] == 'elbo':
        state.update(x=tokens.reshape(B, T), logits=x.to(dt).reshape(B, T, V).requires_grad_(True),
                     kld=(torch.rand(B, generator=g, device=DEV) * 20.0).to(dt).requires_grad_(True), beta=0.5)
        return state
    state.update(tokens=tokens, logits=x.to(dt).requires_grad_(case['op'] == 'policy'))
    if case['op'] == 'policy':
        state['advantage'] = torch.randn(N, generator=g, device=DEV)
        state['bonus'] = torch.rand(N, generator=g, device=DEV) * 0.02
    return state


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(state):
    case = state['case']
    if own:
        return _own(case, state)
    with torch.no_grad():
        if case['op'] == 'score':
            return _plain_score(state['logits'], state['tokens'], case['k'], case['entropy'])
        if case['op'] == 'policy':
            return _plain_policy(state, case['entropy'])
        if case['op'] == 'elbo':
            return _plain_elbo(state)
        return _plain_distill(case, state)


def _own(case, state):
    import vae_amd
    from vae_amd import functional as F_
    if case['op'] == 'score':
        with torch.no_grad():
            lp, ent, top, ids = F_.token_log_probs(state['logits'], state['tokens'], top_k=case['k'],
                                                   want_entropy=case['entropy'])
        out = {'log_prob': lp}
        if case['entropy']:
            out['entropy'] = ent
        if case['k']:
            out['top'], out['ids'] = top, ids
        return out
    if case['op'] == 'policy':
        lp, ent, _, _ = F_.token_log_probs(state['logits'], state['tokens'], want_entropy=case['entropy'])
        if case['entropy']:
            grad, = torch.autograd.grad([lp, ent], [state['logits']], [state['advantage'], state['bonus']])
            return {'log_prob': lp.detach(), 'entropy': ent.detach(), 'grad': grad}
        grad, = torch.autograd.grad([lp], [state['logits']], [state['advantage']])
        return {'log_prob': lp.detach(), 'grad': grad}
    if case['op'] == 'elbo':
        out = vae_amd.loss_function(state['logits'], state['x'], state['kld'], 'categorical', kl_beta=state['beta'])
        grad, gkld = torch.autograd.grad([out['loss_mean']], [state['logits'], state['kld']])
        return {'loss': out['loss'].detach(), 'elbo': out['elbo'].detach(), 'loss_mean': out['loss_mean'].detach(),
                'nll_mean': out['nll_mean'].detach(), 'grad': grad, 'grad_kld': gkld}
    inv = 1.0 / _live_count(case)
    if case['how'] == 'eval':
        with torch.no_grad():
            kl, mean = F_.distill_top_logits(state['logits'], state['teacher'], state['ids'],
                                             temperature=case['tau'], inv_count=inv)
        return {'kl': kl, 'mean': mean}
    kl, mean = F_.distill_top_logits(state['logits'], state['teacher'], state['ids'], temperature=case['tau'],
                                     inv_count=inv, fuse_backward=case['how'] == 'mean')
    if case['how'] == 'mean':
        grad, = torch.autograd.grad([mean], [state['logits']])
    else:
        grad, = torch.autograd.grad([kl], [state['logits']], [state['weights']])
    return {'kl': kl.detach(), 'mean': mean.detach(), 'grad': grad}


# ---- the plain forms: float32, rounded at the end ---------------------------------------------------------------------
def _plain_softmax(x):
    """x [N, V] float32 -> (x - max, exp of it, its sum, log-sum-exp without the maximum)."""
    m = x.amax(-1, keepdim=True)
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    d = x - m
    e = torch.exp(d)
    s = e.sum(-1, keepdim=True)
    return d, e, s, torch.log(s)


def _plain_log_prob(d, s, logs, tokens):
    pad = tokens < 0
    lp = d.gather(1, tokens.clamp(min=0)[:, None])[:, 0] - logs[:, 0]
    lp = torch.where(s[:, 0] == 0, torch.full_like(lp, float('-inf')), lp)
    return torch.where(pad, torch.zeros_like(lp), lp), pad


def _plain_entropy(d, e, s, logs, pad):
    h = logs[:, 0] - (d.clamp(min=-1e4) * e).sum(-1) / s[:, 0]
    return torch.where(pad | (s[:, 0] == 0), torch.zeros_like(h), h)


def _plain_score(logits, tokens, k, want_entropy):
    x = logits.float()
    d, e, s, logs = _plain_softmax(x)
    lp, pad = _plain_log_prob(d, s, logs, tokens)
    out = {'log_prob': lp}
    if want_entropy:
        out['entropy'] = _plain_entropy(d, e, s, logs, pad)
    if k:
        # value first, then the lower index: both in one sortable integer
        bits = (x + 0.0).view(torch.int32)
        order = (bits ^ ((bits >> 31) & 0x7fffffff)).long()
        key = (order << 32) + (0xffffffff - torch.arange(x.shape[1], device=x.device))
        ids = 0xffffffff - (key.topk(k, dim=-1)[0] & 0xffffffff)
        top = d.gather(1, ids) - logs
        out['top'] = torch.where(pad[:, None], torch.full_like(top, float('-inf')), top)
        out['ids'] = torch.where(pad[:, None], torch.full_like(ids, -1), ids)
    return out


def _plain_policy(state, want_entropy):
    logits, tokens = state['logits'], state['tokens']
    d, e, s, logs = _plain_softmax(logits.float())
    lp, pad = _plain_log_prob(d, s, logs, tokens)
    p = e / s
    a = torch.where(pad, torch.zeros_like(lp), state['advantage'])
    grad = -a[:, None] * p
    out = {'log_prob': lp}
    if want_entropy:
        h = _plain_entropy(d, e, s, logs, pad)
        b = torch.where(pad, torch.zeros_like(lp), state['bonus'])
        grad = grad - b[:, None] * p * ((d - logs).clamp(min=-1e4) + h[:, None])
        out['entropy'] = h
    grad.scatter_add_(1, tokens.clamp(min=0)[:, None], a[:, None])
    out['grad'] = grad.to(logits.dtype)
    return out


def _plain_elbo(state):
    B, T, V = state['logits'].shape
    dt = state['logits'].dtype
    tokens = state['x'].reshape(-1)
    d, e, s, logs = _plain_softmax(state['logits'].reshape(-1, V).float())
    lp, pad = _plain_log_prob(d, s, logs, tokens)
    nll = -lp.reshape(B, T).sum(-1)
    kld = state['kld'].float()
    loss, elbo = nll + state['beta'] * kld, nll + kld
    c = torch.where(pad, 0.0, 1.0 / B)
    grad = c[:, None] * (e / s)
    grad.scatter_add_(1, tokens.clamp(min=0)[:, None], -c[:, None])
    return {'loss': loss.to(dt), 'elbo': elbo.to(dt), 'loss_mean': loss.mean().to(dt), 'nll_mean': nll.mean().to(dt),
            'grad': grad.reshape(B, T, V).to(dt), 'grad_kld': torch.full_like(kld, state['beta'] / B).to(dt)}


def _plain_distill(case, state):
    logits, ids = state['logits'], state['ids'].long()
    here = ids >= 0
    at = ids.clamp(min=0)
    tau = case['tau']
    d, e, s, logs = _plain_softmax(logits.float() / tau)
    y = (state['teacher'].float() / tau).masked_fill(~here, float('-inf'))
    yd, ye, ys, ylogs = _plain_softmax(y)
    some = ys > 0
    q = torch.where(some, ye / ys, torch.zeros_like(ye))
    logq = torch.where(q > 0, yd - ylogs, torch.zeros_like(yd))
    logp = torch.where(q > 0, d.gather(1, at) - logs, torch.zeros_like(yd))
    kl = (q * (logq - logp)).sum(-1)
    inv = 1.0 / _live_count(case)
    out = {'kl': kl, 'mean': kl.sum() * inv}
    if case['how'] != 'eval':
        w = torch.full_like(kl, inv) if case['how'] == 'mean' else state['weights']
        w = torch.where(some, w[:, None] / tau, torch.zeros_like(ys))
        grad = w * (e / s)
        grad.scatter_add_(1, at, -w * q)
        out['grad'] = grad.to(logits.dtype)
    return out


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in float64
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        z = state['logits'].detach().double().reshape(-1, case['V'])
        if case['op'] == 'distill':
            return _exact_distill(case, state, z)
        tokens = state['tokens' if 'tokens' in state else 'x'].reshape(-1)
        live = tokens >= 0
        logp = torch.log_softmax(z, -1)
        row = torch.arange(z.shape[0], device=DEV)
        lp = torch.where(live, logp[row, tokens.clamp(min=0)], 0.0)
        p = logp.exp()
        if case['op'] == 'elbo':
            nll = -lp.reshape(case['B'], case['T']).sum(1)
            kld = state['kld'].detach().double()
            loss = nll + 0.5 * kld
            p[row, tokens.clamp(min=0)] -= 1.0
            grad = (p * (live.double() / case['B'])[:, None]).reshape(state['logits'].shape)
            return {'loss': loss, 'elbo': nll + kld, 'loss_mean': loss.mean(), 'nll_mean': nll.mean(), 'grad': grad,
                    'grad_kld': torch.full_like(kld, 0.5 / case['B'])}
        out = {'log_prob': lp}
        plogp = torch.where(p > 0, p * logp, 0.0)
        h = torch.where(live, -plogp.sum(1), 0.0)
        if case['entropy']:
            out['entropy'] = h
        if case['op'] == 'score':
            if case['k']:
                top = logp.topk(case['k'], dim=1)[0]
                out['top'] = torch.where(live[:, None], top, float('-inf'))
                out['ids'] = None
            return out
        a = torch.where(live, state['advantage'].double(), 0.0)
        grad = p * -a[:, None]
        grad[row, tokens.clamp(min=0)] += a
        if case['entropy']:
            grad -= torch.where(live, state['bonus'].double(), 0.0)[:, None] * (plogp + p * h[:, None])
        out['grad'] = grad
        return out


def _exact_distill(case, state, z):
    tau, ids = case['tau'], state['ids'].long()
    logp = torch.log_softmax(z / tau, -1)
    live = (ids >= 0).all(1)                                   # a row of these cases is whole or padding
    ids = torch.where(live[:, None], ids, 0)
    logq = torch.log_softmax(state['teacher'].double() / tau, -1)
    q = torch.where(live[:, None], logq.exp(), 0.0)
    kl = (q * (logq - logp.gather(1, ids))).sum(1)
    out = {'kl': kl, 'mean': kl.sum() / live.sum()}
    if case['how'] != 'eval':
        w = torch.full_like(kl, 1.0) / live.sum() if case['how'] == 'mean' else state['weights'].double()
        w = torch.where(live, w / tau, 0.0)[:, None]
        out['grad'] = (logp.exp() * w).scatter_add(1, ids, -q * w)
    return out


def work(case):
    """Each live row of logits read once; each output written once."""
    rows, live, V, e = case['B'] * case.get('T', 1), _live_count(case), case['V'], SIZE[case['dtype']]
    read = live * V * e
    if case['op'] == 'score':
        small = rows * (8 + 4 + (4 if case['entropy'] else 0) + 12 * case['k'])
        return {'bytes': read + small, 'flops': live * V * (6 if case['entropy'] else 4)}
    if case['op'] == 'policy':
        return {'bytes': read + rows * V * e + rows * 24, 'flops': live * V * (12 if case['entropy'] else 7)}
    if case['op'] == 'elbo':
        return {'bytes': read + rows * V * e + rows * 8 + case['B'] * 4 * e, 'flops': live * V * 7}
    teacher = rows * case['K'] * (4 + e)
    if case['how'] == 'eval':
        return {'bytes': read + teacher + rows * 4, 'flops': live * V * 4}
    return {'bytes': read + rows * V * e + teacher + rows * 4, 'flops': live * V * 7}
