# -*- coding: utf-8 -*-
"""Cases of the language-model operators: what each computes in plain tensor operations, the calls a user makes of the
package, and what the definition gives in 64 bits.

Kinds of case:

* ``embed``  -- rows of an embedding table times a factor (``mgwfbp_b200.ops.embedding``), and with ``train`` the dense
  gradient of the table: the sum of the rows' gradients for each token;
* ``score``  -- log probability of given tokens, entropy of the distribution and the ``top`` likeliest tokens of every
  row of logits (``mgwfbp_b200.ops.logprob``), and with ``train`` the gradient of the logits for given gradients of log
  probability and entropy;
* ``loss``   -- mean cross entropy over the rows that are not padding, with the gradient of the logits;
* ``clip``   -- global norm of a model's gradients and their scaling to a largest norm, in place
  (``mgwfbp_b200.ops.clip``).
"""
import math

import torch

own = False

DTYPES = {'fp32': torch.float32, 'bf16': torch.bfloat16, 'fp16': torch.float16}
BYTES = {'fp32': 4, 'bf16': 2, 'fp16': 2}
IGNORE = -100
MAX_NORM = 0.25


def listed():
    return [
        # the PTB model predicts one more word for each of its 20 streams: latency is all
        dict(name='embed one step', kind='embed', train=False, tokens=20, vocab=10000, dim=1500, dtype='fp32', scaled=False),
        # the PTB model's training window, 35 steps of 20 streams, with the gradient of its 10000 x 1500 table
        dict(name='embed ptb window', kind='embed', train=True, tokens=700, vocab=10000, dim=1500, dtype='fp32', scaled=False),
        # a ragged batch on a mid-sized half-precision table of odd width, rows scaled by sqrt(dim)
        dict(name='embed ragged', kind='embed', train=True, tokens=20011, vocab=32003, dim=1023, dtype='fp16', scaled=True),
        # a large model's training batch
        dict(name='embed large', kind='embed', train=True, tokens=262144, vocab=131072, dim=2048, dtype='bf16', scaled=True),
        # the next word of 20 streams with its five likeliest alternatives
        dict(name='score one step', kind='score', train=False, rows=20, vocab=10000, pad=0, top=5, dtype='fp32', masked=False),
        # evaluation of one PTB window with per-word statistics
        dict(name='score ptb window', kind='score', train=False, rows=700, vocab=10000, pad=0, top=5, dtype='fp32', masked=False),
        # long prompts scored on an odd vocabulary inside a padded output layer, a tenth of it not allowed
        dict(name='score prompts', kind='score', train=False, rows=4099, vocab=50261, pad=43, top=20, dtype='bf16', masked=True),
        # policy training: gradient of chosen log probabilities and of the entropy
        dict(name='score train', kind='score', train=True, rows=2048, vocab=32000, pad=0, top=0, dtype='bf16', masked=False),
        # the PTB model's loss and its gradient
        dict(name='loss ptb window', kind='loss', rows=700, vocab=10000, pad=0, dtype='fp32', padding=0.0, loss_scale=1.0),
        # a large vocabulary's loss, an eighth of the rows being padding
        dict(name='loss large', kind='loss', rows=8192, vocab=131072, pad=0, dtype='bf16', padding=0.125, loss_scale=1.0),
        # the PTB model's gradients (66 million values in 11 tensors), clipped to 0.25
        dict(name='clip ptb', kind='clip', model='ptb', tensors=11, elements=66034000, dtype='fp32'),
        # many tensors of very different sizes, as a 50-layer convolutional network has them
        dict(name='clip many', kind='clip', model='', tensors=161, elements=25557032, dtype='fp32'),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(['embed', 'score', 'loss', 'clip'])
    dtype = rng.choice(['fp32', 'bf16', 'fp16'])
    if kind == 'embed':
        train = rng.random() < 0.75
        vocab, dim = _log(rng, 1000, 131072), _log(rng, 128, 2048)
        # the cost is rows read, rows written and the dense gradient: all within the largest listed case
        tokens = min(_log(rng, 1, 262144), 262144 * 4096 // (dim * BYTES[dtype]))
        return dict(kind=kind, train=train, tokens=tokens, vocab=vocab, dim=dim, dtype=dtype, scaled=rng.random() < 0.5)
    if kind == 'score':
        vocab = _log(rng, 1000, 131072)
        rows = min(_log(rng, 1, 8192), 8192 * 131072 // 4 // vocab)
        return dict(kind=kind, train=rng.random() < 0.4, rows=rows, vocab=vocab, pad=rng.choice([0, 0, 1, 8, 61]),
                    top=rng.choice([0, 1, 5, 20, 32]), dtype=dtype, masked=rng.random() < 0.3)
    if kind == 'loss':
        vocab = _log(rng, 1000, 131072)
        rows = min(_log(rng, 1, 8192), 8192 * 131072 // (2 * BYTES[dtype]) // vocab)
        return dict(kind=kind, rows=rows, vocab=vocab, pad=rng.choice([0, 0, 1, 8, 61]), dtype=dtype,
                    padding=rng.choice([0.0, 0.0, 0.1, 0.5]), loss_scale=128.0 if dtype == 'fp16' else 1.0)
    tensors = _log(rng, 1, 400)
    return dict(kind=kind, model='', tensors=tensors, elements=max(_log(rng, 1000, 1 << 28), tensors), dtype=dtype)


# ------------------------------------------------------------------------------------------------------------ inputs
def _sizes(case):
    """Element counts of the gradients of a ``clip`` case."""
    if case['model'] == 'ptb':       # embedding, two layers of a 1500-wide LSTM, output layer and bias
        per_layer = [6000 * 1500, 6000 * 1500, 6000, 6000]
        return [10000 * 1500] + per_layer + per_layer + [10000 * 1500, 10000]
    n, total = case['tensors'], case['elements']
    weight = [((i * 7919 + 13) % 101 + 1) ** (1 if i % 3 else 3) for i in range(n)]       # biases between matrices
    whole = sum(weight)
    sizes = [max(1, total * w // whole) for w in weight]
    sizes[sizes.index(max(sizes))] += max(0, total - sum(sizes))
    return sizes


def _zipf(u, vocab):
    """Word ranks with probability about 1 / (rank + 1): ids in order of frequency, as vocabularies are built."""
    return (torch.exp(u * math.log(vocab + 1)) - 1).to(torch.int64).clamp_(0, vocab - 1)


def _logits(case, gen):
    """Rows as an output layer gives them: frequent words likelier, one or two guesses that stand out, and (``masked``) a
    tenth of the vocabulary at minus infinity.  ``pad`` columns behind the vocabulary belong to the layer, not to the
    operator."""
    rows, vocab, dtype = case['rows'], case['vocab'], DTYPES[case['dtype']]
    wide = torch.empty(rows, vocab + case['pad'], dtype=dtype, device='cuda').normal_(0.0, 1.5, generator=gen)
    z = wide[:, :vocab]
    z -= torch.log(torch.arange(2, vocab + 2, device='cuda', dtype=torch.float32)).to(dtype)
    guess = _zipf(torch.rand(rows, device='cuda', generator=gen), vocab)
    lift = torch.rand(rows, device='cuda', generator=gen) * 12
    at = torch.arange(rows, device='cuda')
    z[at, guess] += lift.to(dtype)
    if case.get('masked'):
        off = torch.rand(vocab, device='cuda', generator=gen) < 0.1
        z.masked_fill_(off, float('-inf'))
        z[at, guess] = lift.to(dtype)
    other = _zipf(torch.rand(rows, device='cuda', generator=gen), vocab)
    hit = torch.rand(rows, device='cuda', generator=gen) < 0.6
    if case.get('masked'):
        other = guess                     # a chosen token is one that was allowed
    tokens = torch.where(hit, guess, other)
    if case.get('padding'):
        tokens = tokens.masked_fill(torch.rand(rows, device='cuda', generator=gen) < case['padding'], IGNORE)
        tokens[0] = guess[0]
    return z, tokens


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    dtype, kind = DTYPES[case['dtype']], case['kind']
    state = dict(case=case)
    if kind == 'embed':
        n, vocab, dim = case['tokens'], case['vocab'], case['dim']
        shape = (35, 20) if n == 700 else (n,)
        state['tokens'] = _zipf(torch.rand(n, device='cuda', generator=gen), vocab).view(shape)
        state['scale'] = math.sqrt(dim) if case['scaled'] else 1.0
        weight = torch.empty(vocab, dim, dtype=dtype, device='cuda').uniform_(-0.1, 0.1, generator=gen)
        state['weight'] = weight.requires_grad_(case['train'])
        if case['train']:
            state['grad'] = torch.empty(*shape, dim, dtype=dtype, device='cuda').normal_(0.0, 0.02, generator=gen)
    elif kind in ('score', 'loss'):
        z, state['tokens'] = _logits(case, gen)
        train = kind == 'loss' or case['train']
        state['logits'] = z.detach().requires_grad_(train)
        if kind == 'score' and train:
            state['grad_logprob'] = torch.empty(case['rows'], device='cuda').normal_(0.0, 1.0, generator=gen)
            state['grad_entropy'] = torch.full((case['rows'],), 0.01, device='cuda')
        if kind == 'loss':                # half-precision training scales its loss
            state['upstream'] = torch.tensor(case['loss_scale'], device='cuda')
    else:
        sizes = _sizes(case)
        flat = torch.empty(sum(sizes), dtype=dtype, device='cuda').normal_(0.0, 0.01, generator=gen)
        state['flat'], state['params'], at = flat, [], 0
        for n in sizes:                   # gradients that live in one merged buffer, one tensor behind the other
            p = torch.nn.Parameter(torch.empty(n, dtype=dtype, device='cuda'))
            p.grad = flat[at:at + n]
            state['params'].append(p)
            at += n
    return state


# --------------------------------------------------------------------------------------------------------- operators
def run(state):
    kind = state['case']['kind']
    if kind == 'embed':
        return _run_embed(state)
    if kind == 'score':
        return _run_score(state)
    if kind == 'loss':
        return _run_loss(state)
    return _run_clip(state)


def _run_embed(s):
    tokens, weight, scale, train = s['tokens'], s['weight'], s['scale'], s['case']['train']
    if own:
        from mgwfbp_b200.ops.embedding import embedding
        out = embedding(tokens, weight, scale=scale)
        if not train:
            return out
        (dw,) = torch.autograd.grad(out, weight, s['grad'])
        return out, dw
    w = weight.detach()
    out = (w[tokens].float() * scale).to(w.dtype)
    if not train:
        return out
    dw = torch.zeros(w.shape, dtype=torch.float32, device=w.device)
    dw.index_add_(0, tokens.reshape(-1), s['grad'].reshape(-1, w.shape[1]).float())
    return out, (dw * scale).to(w.dtype)


def _run_score(s):
    case, z, tokens = s['case'], s['logits'], s['tokens']
    if own:
        from mgwfbp_b200.ops.logprob import token_log_probs
        r = token_log_probs(z, tokens, top=case['top'])
        out = [r.logprob, r.entropy] + ([r.top_logprob, r.top_tokens] if case['top'] else [])
        if case['train']:
            out += torch.autograd.grad([r.logprob, r.entropy], [z], [s['grad_logprob'], s['grad_entropy']])
        return out
    x = z.detach().float()
    d = x - x.amax(1, keepdim=True)
    e = d.exp()
    total = e.sum(1, keepdim=True)
    logp = d - total.log()
    p = e / total
    surprise = torch.where(e > 0, logp, 0.0)                # a probability of zero adds nothing to the entropy
    entropy = -(p * surprise).sum(1)
    chosen = tokens.unsqueeze(1)
    out = [logp.gather(1, chosen).squeeze(1), entropy]
    if case['top']:
        bits = (x + 0.0).view(torch.int32)                  # whole numbers in the order of the values, then the lower index
        order = torch.where(bits < 0, bits ^ 0x7fffffff, bits).to(torch.int64)
        key = (order << 32) + (0xffffffff - torch.arange(case['vocab'], device=x.device))
        best = 0xffffffff - (key.topk(case['top'], dim=1).values & 0xffffffff)
        out += [logp.gather(1, best), best]
    if case['train']:
        g1, g2 = s['grad_logprob'].unsqueeze(1), s['grad_entropy'].unsqueeze(1)
        dz = -p * (g1 + g2 * (surprise + entropy.unsqueeze(1)))
        dz.scatter_add_(1, chosen, g1)
        out.append(dz.to(z.dtype))
    return out


def _run_loss(s):
    z, tokens = s['logits'], s['tokens']
    if own:
        from mgwfbp_b200.ops.logprob import cross_entropy
        loss = cross_entropy(z, tokens, ignore_index=IGNORE, expected_grad=s['case']['loss_scale'])
        return (loss,) + torch.autograd.grad(loss, z, s['upstream'])
    x = z.detach().float()
    d = x - x.amax(1, keepdim=True)
    e = d.exp()
    total = e.sum(1, keepdim=True)
    keep = tokens != IGNORE
    count = keep.sum()
    chosen = torch.where(keep, tokens, 0).unsqueeze(1)
    logp = (d.gather(1, chosen) - total.log()).squeeze(1)
    loss = -(torch.where(keep, logp, 0.0).sum() / count)
    factor = (s['upstream'] * keep / count).unsqueeze(1)
    dz = e * (factor / total)
    dz.scatter_add_(1, chosen, -factor)
    return loss, dz.to(z.dtype)


def _run_clip(s):
    # the factor: gradients were averaged over two ranks, and this user's step size is set for their sum
    if own:
        from mgwfbp_b200.ops.clip import clip_grad_norm_
        return clip_grad_norm_(s['params'], MAX_NORM, grad_scale=2.0), s['flat']
    g = s['flat'].float()                                   # every tensor at once: they lie one behind the other
    norm = (g * 2.0).square().sum().sqrt()
    g *= 2.0 * (MAX_NORM / (norm + 1e-6)).clamp(max=1.0)
    return norm, s['flat'].copy_(g)


# -------------------------------------------------------------------------------------------------------------- work
def work(case):
    kind, size = case['kind'], BYTES[case['dtype']]
    if kind == 'embed':
        n, vocab, dim = case['tokens'], case['vocab'], case['dim']
        rank = torch.arange(1, vocab + 1, dtype=torch.float64)
        p = torch.log1p(1.0 / rank) / math.log(vocab + 1)
        distinct = float((1.0 - (1.0 - p) ** n).sum())                # rows of the table that have to be read
        moved = n * 8 + (distinct + n) * dim * size
        if case['train']:
            moved += n * 8 + (n + vocab) * dim * size
        return dict(bytes=moved, flops=float(n * dim * (2 if case['train'] else 1)))
    if kind == 'clip':
        return dict(bytes=2 * case['elements'] * size + 4, flops=3.0 * case['elements'])
    cells = case['rows'] * case['vocab']
    if kind == 'loss':
        return dict(bytes=2 * cells * size + case['rows'] * 8 + 4, flops=6.0 * cells)
    moved = cells * size + case['rows'] * (8 + 8 + case['top'] * 12)
    if case['train']:
        moved += cells * size + case['rows'] * 8
    return dict(bytes=moved, flops=(12.0 if case['train'] else 6.0) * cells)


# ------------------------------------------------------------------------------------------------- values in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case['kind'] == 'embed':
        ids = s['tokens']
        out = torch.nn.functional.embedding(ids, s['weight'].detach().double()).mul_(s['scale'])
        if not case['train']:
            return out
        order = torch.argsort(ids.reshape(-1), stable=True)
        dw = torch.zeros(case['vocab'], case['dim'], dtype=torch.float64, device='cuda')
        g = s['grad'].reshape(-1, case['dim'])
        for piece in order.split(1 << 16):
            dw.index_put_((ids.reshape(-1)[piece],), g[piece].double() * s['scale'], accumulate=True)
        return out, dw
    if case['kind'] == 'clip':
        g = 2.0 * s['flat'].double()
        norm = torch.linalg.vector_norm(g)
        if norm + 1e-6 > MAX_NORM:
            g *= MAX_NORM / (norm + 1e-6)
        return norm, g
    step = max(1, (1 << 27) // case['vocab'])                          # rows at a time: at most 1 GB of 64-bit values
    parts = [_exact_rows(case, s, slice(a, a + step)) for a in range(0, case['rows'], step)]
    joined = [torch.cat(v) if isinstance(v[0], torch.Tensor) else None for v in zip(*parts)]
    if case['kind'] == 'loss':
        kept = (s['tokens'] != IGNORE).sum()
        return joined[0].sum() / kept, joined[1] * case['loss_scale']
    return joined


def _exact_rows(case, s, rows):
    z = s['logits'].detach()[rows].double()
    lse = torch.logsumexp(z, 1)
    tokens = s['tokens'][rows]
    at = torch.arange(len(z), device=z.device)
    prob = torch.softmax(z, 1)
    if case['kind'] == 'loss':
        count = (s['tokens'] != IGNORE).sum()
        valid = tokens != IGNORE
        loss = torch.where(valid, lse - z[at, tokens.clamp(min=0)], 0.0)
        prob[at[valid], tokens[valid]] -= 1.0
        prob *= valid.double().unsqueeze(1) / count
        return loss, prob
    entropy = torch.special.entr(prob).sum(1)
    out = [z[at, tokens] - lse, entropy]
    if case['top']:
        value, index = torch.sort(z, dim=1, descending=True, stable=True)
        out += [value[:, :case['top']] - lse.unsqueeze(1), index[:, :case['top']].clone()]
    if case['train']:
        g1, g2 = (s[k][rows].double() for k in ('grad_logprob', 'grad_entropy'))
        log_prob = torch.log_softmax(z, 1).nan_to_num(neginf=0.0)
        dz = prob.mul(-1.0) * (g1[:, None] + g2[:, None] * (log_prob + entropy[:, None]))
        dz[at, tokens] += g1
        out.append(dz)
    return out
