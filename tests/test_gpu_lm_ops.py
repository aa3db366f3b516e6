"""Embedding, token log probabilities, cross entropy and gradient clipping on the GPU against 64-bit evaluations, with the
bounds that ``lm_oracle`` derives."""
import math

import pytest
import torch

from lm_oracle import Rows, U, assert_within, embedding_grad as oracle_grad, half_step, tiny

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
ids = lambda v: str(v).replace('torch.', '') if isinstance(v, torch.dtype) else None      # noqa: E731


def _tokens(kind, n, vocab, gen):
    if kind == 'same':
        return torch.full((n,), vocab // 2, device='cuda')
    if kind == 'zipf':
        u = torch.rand(n, device='cuda', generator=gen)
        return (torch.exp(u * math.log(vocab + 1)) - 1).long().clamp_(0, vocab - 1)
    if kind == 'last':
        return torch.full((n,), vocab - 1, device='cuda')
    return torch.randint(0, vocab, (n,), device='cuda', generator=gen)


# ---------------------------------------------------------------------------------------------------------- embedding
@pytest.mark.parametrize('dtype', TYPES, ids=ids)
@pytest.mark.parametrize('n,vocab,dim,kind', [
    (1, 1, 1, 'any'), (1, 10, 4, 'any'), (2, 3, 7, 'same'), (7, 5, 33, 'any'), (31, 100, 128, 'last'), (33, 2, 130, 'any'),
    (700, 1000, 1500, 'zipf'), (2047, 257, 1023, 'zipf'), (2049, 70000, 8, 'any'), (4099, 33, 258, 'zipf'), (5000, 300, 640, 'same'),
    (20011, 5003, 129, 'zipf'), (40000, 131072, 24, 'zipf')])
def test_embedding_forward_and_gradient(n, vocab, dim, kind, dtype):
    from mgwfbp_b200.ops.embedding import check_status, embedding
    gen = torch.Generator(device='cuda').manual_seed(n)
    t = _tokens(kind, n, vocab, gen)
    t = t.int() if n % 2 else t
    w = torch.randn(vocab, dim, device='cuda', generator=gen).to(dtype).requires_grad_()
    for scale, padding in ((1.0, None), (math.sqrt(dim) + 0.1, int(t[0]))):
        out = embedding(t, w, scale, padding)
        want = w.detach()[t.long()].double() * scale
        if scale == 1.0:
            assert torch.equal(out, w.detach()[t.long()])
        # the factor and the product round in fp32, the result to the type
        assert_within(out, want, want.abs() * (half_step(dtype) + 2.001 * U) + tiny(dtype), 'out')
        dy = torch.randn(n, dim, device='cuda', generator=gen).to(dtype)
        (dw,) = torch.autograd.grad(out, w, dy)
        want, bound = oracle_grad(dy, t, vocab, scale, padding)
        assert_within(dw, want, bound, 'dw')
        (again,) = torch.autograd.grad(embedding(t, w, scale, padding), w, dy)
        assert torch.equal(dw, again)                                            # the same on every run
    check_status()


@pytest.mark.parametrize('dtype', TYPES, ids=ids)
def test_embedding_every_width_and_alignment(dtype):
    """Rows that begin and end anywhere in a 16-byte block, in the table, the output, the gradient and its sum; short lists
    (one launch), longer ones, and ones that leave most rows without a token."""
    from mgwfbp_b200.ops.embedding import embedding, embedding_grad
    gen = torch.Generator(device='cuda').manual_seed(7)
    store = torch.randn(4, 41, 600, device='cuda', generator=gen).to(dtype)
    for dim in list(range(1, 41)) + [63, 64, 65, 127, 128, 129, 255, 256, 257, 258, 383, 511, 512, 513, 590]:
        for at in range(0, 8 if dim < 41 else 3):
            w = store[dim % 4, :, at:at + dim]                       # rows 600 apart, from any element
            for n in (5, 1500):
                t = torch.randint(0, 41, (n,), device='cuda', generator=gen)
                assert torch.equal(embedding(t, w), w[t]), (dim, at, n)
                wide = torch.randn(n, dim + at + 3, device='cuda', generator=gen).to(dtype)
                dy = wide[:, at:at + dim]
                want, bound = oracle_grad(dy, t, 43, 1.0)
                assert_within(embedding_grad(dy, t, 43), want, bound, 'dw %d %d %d' % (dim, at, n))


def test_embedding_gradient_writes_nothing_else():
    """The rows behind and before the result stay as they were."""
    from mgwfbp_b200.ops import _lib
    from mgwfbp_b200.ops._tokens import status_words
    lib = _lib.load(allow_build=False)
    for n in (6, 3000, 70000):
        for dim, shift in ((37, 3), (64, 0)):
            t = torch.randint(0, 50, (n,), device='cuda')
            dy = torch.randn(n, dim, device='cuda')
            store = torch.full((60 * dim + 16,), 7.0, device='cuda')
            dw = store[5 * dim + shift:55 * dim + shift]
            need = lib.mgw_embedding_grad_bytes(n, 50, dim, 0)
            work = torch.empty(need, dtype=torch.uint8, device='cuda')
            assert lib.mgw_embedding_grad(dy.data_ptr(), dim, t.data_ptr(), 1, n, 50, dim, 0, 1.0, -1, None, dw.data_ptr(),
                                          work.data_ptr() if need else None, need, status_words(),
                                          torch.cuda.current_stream().cuda_stream) == 0
            want, bound = oracle_grad(dy, t, 50, 1.0)
            assert_within(dw.view(50, dim), want, bound, 'dw')
            assert (store[:5 * dim + shift] == 7).all() and (store[55 * dim + shift:] == 7).all()


def test_embedding_strides_shapes_and_broadcast_gradient():
    from mgwfbp_b200.ops.embedding import embedding, embedding_grad
    wide = torch.randn(50, 40, device='cuda')
    t = torch.randint(0, 50, (6, 8), device='cuda').t()                          # not contiguous
    for cols in (slice(0, 32), slice(1, 33), slice(3, 20)):                      # rows further apart, odd starts
        w = wide[:, cols].detach().requires_grad_()
        out = embedding(t, w)
        assert out.shape == (8, 6, w.shape[1]) and torch.equal(out, w.detach()[t])
        (dw,) = torch.autograd.grad(out.sum(), w)                                # a gradient of stride zero
        want = torch.bincount(t.reshape(-1), minlength=50).float().unsqueeze(1).expand(50, w.shape[1])
        assert torch.equal(dw, want)
    dy = torch.randn(8, 6, 96, device='cuda')[..., 5:69]
    want, bound = oracle_grad(dy, t, 50, 1.0)
    assert_within(embedding_grad(dy, t, 50), want, bound, 'strided dy')
    w = wide.t().detach().requires_grad_()                                       # columns of another matrix
    t2 = torch.tensor([0, 39, 39], device='cuda')
    out = embedding(t2, w, 3.0)
    assert_within(out, w.detach()[t2].double() * 3, out.double().abs() * 2 * U, 'transposed table')


@pytest.mark.parametrize('n', [5, 3000, 9000])
def test_embedding_nan_stays_in_its_row(n):
    from mgwfbp_b200.ops.embedding import embedding_grad
    t = torch.arange(n, device='cuda') % 100
    dy = torch.ones(n, 20, device='cuda')
    dy[4] = math.nan                                                             # token 4
    dw = embedding_grad(dy, t, 101, padding_idx=4)
    assert torch.isfinite(dw).all() and not dw[4].any() and not dw[100].any()
    dw = embedding_grad(dy, t, 101)
    assert dw[4].isnan().all() and torch.isfinite(dw[:4]).all() and torch.isfinite(dw[5:]).all()


@pytest.mark.parametrize('n', [6, 5000])
def test_token_outside_the_vocabulary_is_reported(n):
    from mgwfbp_b200.ops import embedding as emb, logprob as lp
    w = torch.randn(10, 12, device='cuda')
    t = torch.arange(n, device='cuda') % 10
    emb.check_status()
    for bad in (10, -1, 1 << 40):
        t[3] = bad
        out = emb.embedding(t, w)
        assert out[3].isnan().all() and torch.equal(out[:3], w[t[:3]]) and torch.equal(out[4:], w[t[4:]])
        with pytest.raises(emb.TokenIndexError, match='position 3'):
            emb.check_status()
        dw = emb.embedding_grad(torch.ones(n, 12, device='cuda'), t, 10)
        with pytest.raises(emb.TokenIndexError, match='gradient'):
            emb.check_status()
        ok = torch.cat([t[:3], t[4:]])
        assert torch.equal(dw, torch.bincount(ok, minlength=10).float().unsqueeze(1).expand(10, 12))
        z = torch.randn(n, 10, device='cuda', requires_grad=True)
        r = lp.token_log_probs(z, t)
        assert r.logprob[3].isnan() and torch.isfinite(r.logprob[:3]).all() and torch.isfinite(r.entropy).all()
        with pytest.raises(lp.TokenIndexError, match='log prob'):
            lp.check_status()
        (dz,) = torch.autograd.grad(r.logprob.sum(), z)
        assert dz[3].isnan().all() and torch.isfinite(dz[:3]).all() and torch.isfinite(dz[4:]).all()
        assert lp.cross_entropy(z, t).isnan()
        with pytest.raises(lp.TokenIndexError):
            lp.check_status()
    emb.check_status()


def test_embedding_offsets_beyond_32_bits():
    from mgwfbp_b200.ops.embedding import embedding, embedding_grad
    w = torch.zeros(70000, 65536, dtype=torch.bfloat16, device='cuda')           # 4.6e9 elements
    w[69999, :] = 3.0
    w[40000, 5] = 2.0
    out = embedding(torch.tensor([69999, 40000, 0], device='cuda'), w)
    assert (out[0] == 3).all() and out[1, 5] == 2 and out[1].sum() == 2 and not out[2].any()
    del w
    dw = embedding_grad(out, torch.tensor([69999, 40000, 69999], device='cuda'), 70000)
    assert (dw[69999] == 3).all() and dw[40000, 5] == 2 and dw[40000].sum() == 2
    dw[69999] = 0
    dw[40000] = 0
    assert not dw.any()


# ----------------------------------------------------------------------------------------------------- log probabilities
def _case(rows, vocab, pad, dtype, seed, special=True):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    wide = (torch.randn(rows, vocab + pad, device='cuda', generator=gen) * 4).to(dtype)
    z = wide[:, :vocab]
    t = torch.randint(0, vocab, (rows,), device='cuda', generator=gen)
    if special:
        low = torch.finfo(dtype).min
        for r in range(rows):
            k = r % 12
            keep = int(t[r])
            if k == 1:                                     # only a few tokens allowed
                z[r, torch.rand(vocab, device='cuda', generator=gen) < 0.9] = -math.inf
                z[r, keep] = 1.0
            elif k == 2:                                   # masked with the type's lowest value
                z[r, torch.rand(vocab, device='cuda', generator=gen) < 0.5] = low
                z[r, keep] = 0.5
            elif k == 3:
                z[r] = 1.5                                 # all equal
            elif k == 4:
                t[r] = -100
                z[r] = math.nan                            # padding: never read
            elif k == 5:
                z[r] = -math.inf                           # nothing left
            elif k == 6:
                z[r, keep] = math.nan
            elif k == 7:
                z[r, vocab // 2] = math.inf
            elif k == 8:
                z[r] = low                                 # all at the lowest value: all equal
            elif k == 9:
                z[r] = -math.inf
                z[r, keep] = -3.0                          # one token left
            elif k == 10:
                z[r] += 500.0                              # far from zero
            elif k == 11:
                z[r] = z[r].abs() * 0.0                    # zeros of both signs
                z[r, ::2] *= -1.0
    return z, t


SHAPES = [(1, 1, 0), (3, 2, 0), (13, 31, 1), (13, 127, 0), (12, 128, 0), (26, 1000, 0), (12, 1024, 8), (24, 10000, 0), (25, 10001, 0),
          (13, 50261, 43), (12, 32768, 0), (12, 131072, 0), (1, 100003, 0)]


@pytest.mark.parametrize('dtype', TYPES, ids=ids)
@pytest.mark.parametrize('rows,vocab,pad', SHAPES)
def test_log_probs_and_gradient(rows, vocab, pad, dtype):
    from mgwfbp_b200.ops.logprob import check_status, token_log_probs
    z, t = _case(rows, vocab, pad, dtype, rows * 7 + vocab)
    z = z.detach().requires_grad_()
    want = Rows(z, t)
    for top in sorted({0, 1, min(5, vocab), min(20, vocab), min(32, vocab)}):
        r = token_log_probs(z, t if top % 2 else t.int(), top=top)
        assert_within(r.logprob, *want.logprob(), 'logprob')
        assert_within(r.entropy, *want.entropy(), 'entropy')
        if top == 0:
            assert r.top_logprob is None and r.top_tokens is None
            continue
        v, bound, order = want.top(top)
        assert torch.equal(r.top_tokens, order), top
        assert_within(r.top_logprob, v, bound, 'top')
    g1, g2 = torch.randn(rows, device='cuda'), torch.randn(rows, device='cuda')
    zero = torch.zeros(rows, device='cuda')
    for outs, gs, ws in (([r.logprob, r.entropy], [g1, g2], (g1, g2)), ([r.logprob], [g1], (g1, zero)), ([r.entropy], [g2], (zero, g2))):
        (dz,) = torch.autograd.grad(outs, [z], gs, retain_graph=True)
        assert dz.dtype == dtype
        w, bound = want.grad(*ws, dtype)
        assert_within(dz, w, bound, 'dz')
    check_status()


@pytest.mark.parametrize('dtype', TYPES, ids=ids)
@pytest.mark.parametrize('rows,vocab,pad', SHAPES)
@pytest.mark.parametrize('reduction,upstream', [('mean', 1.0), ('mean', 128.0), ('sum', -0.37)])
def test_cross_entropy_and_gradient(rows, vocab, pad, dtype, reduction, upstream):
    from mgwfbp_b200.ops.logprob import check_status, cross_entropy
    z, t = _case(rows, vocab, pad, dtype, rows * 11 + vocab, special=False)
    if rows > 2:
        t[1::3] = -100
    z = z.detach().requires_grad_()
    want = Rows(z, t)
    lp, bound = want.logprob()
    n = int((t != -100).sum()) if reduction == 'mean' else 1
    for expected in (1.0, upstream):
        loss = cross_entropy(z, t, reduction=reduction, expected_grad=expected)
        assert loss.dtype == torch.float32 and loss.dim() == 0
        # the rows' errors, and one rounding of the 64-bit sum
        assert_within(loss, -lp.sum() / n, bound[t != -100].sum() / n + U * (lp.sum().abs() / n) * 1.01, 'loss')
        up = torch.tensor(upstream, device='cuda')
        (dz,) = torch.autograd.grad(loss, z, up, retain_graph=True)
        g = torch.full((rows,), -upstream / n, dtype=torch.float64, device='cuda')
        w, b = want.grad(g, torch.zeros_like(g), dtype)
        assert_within(dz, w, b, 'dz')
        (again,) = torch.autograd.grad(loss, z, up)                              # a graph that was kept
        assert torch.equal(dz, again)
    check_status()


def test_cross_entropy_special_rows():
    from mgwfbp_b200.ops.logprob import FusedCrossEntropyLoss, cross_entropy
    z, t = _case(12, 500, 0, torch.float32, 5)
    want = Rows(z, t)
    lp, bound = want.logprob()
    assert_within(cross_entropy(z, t, reduction='none'), -lp, bound, 'none')
    fine = want.fine & ~want.pad
    zz = z.detach().clone().requires_grad_()
    t2 = torch.where(fine | want.pad, t, torch.full_like(t, -100))              # the rows without a distribution become padding
    loss = FusedCrossEntropyLoss()(zz, t2)
    loss.backward()
    ref = z.detach()[fine].double().requires_grad_()
    torch.nn.functional.cross_entropy(ref, t[fine]).backward()
    assert not zz.grad[~fine].any()
    torch.testing.assert_close(zz.grad[fine].double(), ref.grad, rtol=1e-4, atol=1e-6)
    every = torch.full_like(t, -100)
    zz.grad = None
    loss = cross_entropy(zz, every)
    loss.backward()
    assert loss.isnan() and not zz.grad.any()
    assert cross_entropy(zz, every, reduction='sum') == 0


def test_gradients_against_differences():
    """Directional derivative by central differences of the 64-bit functions."""
    from mgwfbp_b200.ops.logprob import token_log_probs
    z, t = _case(6, 301, 0, torch.float32, 3, special=False)
    z = z.detach().requires_grad_()
    r = token_log_probs(z, t)
    (dz,) = torch.autograd.grad((r.logprob + 0.5 * r.entropy).sum(), z)
    v = torch.randn_like(z).double()
    f = lambda s: sum(float(x.sum()) * k for x, k in ((Rows(z.detach().double() + s * v, t).logprob()[0], 1.0),      # noqa: E731
                                                      (Rows(z.detach().double() + s * v, t).entropy()[0], 0.5)))
    got, want = float((dz.double() * v).sum()), (f(1e-5) - f(-1e-5)) / 2e-5
    assert abs(got - want) <= 1e-4 * max(1.0, float((dz.double() * v).abs().sum()))


@pytest.mark.parametrize('dtype', TYPES, ids=ids)
def test_log_probs_every_width_and_alignment(dtype):
    """Vocabularies around the sizes of a vector, a batch, a block and a cluster's parts, rows that begin anywhere."""
    from mgwfbp_b200.ops.logprob import cross_entropy, token_log_probs
    gen = torch.Generator(device='cuda').manual_seed(9)
    widths = list(range(1, 36)) + [k + d for k in (128, 512, 1024, 2048, 4096, 8192, 16384) for d in (-1, 0, 1, 5)]
    for v in widths:
        for rows, at in ((3, v % 8), (2, (v + 3) % 8)):
            wide = (torch.randn(rows, v + 9, device='cuda', generator=gen) * 3).to(dtype)
            z = wide[:, at:at + v].detach().requires_grad_()
            t = torch.randint(0, v, (rows,), device='cuda', generator=gen)
            top = min(7, v)
            want = Rows(z, t)
            r = token_log_probs(z, t, top=top)
            assert_within(r.logprob, *want.logprob(), 'logprob %d' % v)
            assert_within(r.entropy, *want.entropy(), 'entropy %d' % v)
            assert torch.equal(r.top_tokens, want.top(top)[2]), v
            g1, g2 = torch.randn(rows, device='cuda', generator=gen), torch.randn(rows, device='cuda', generator=gen)
            (dz,) = torch.autograd.grad([r.logprob, r.entropy], [z], [g1, g2])
            assert_within(dz, *want.grad(g1, g2, dtype), 'dz %d' % v)
            (dz,) = torch.autograd.grad(cross_entropy(z, t), z)
            assert_within(dz, *want.grad(-torch.ones(rows, device='cuda') / rows, g2 * 0, dtype), 'dloss %d' % v)


@pytest.mark.parametrize('rows', [2, 700])
def test_top_of_sorted_rows_and_ties(rows):
    """Rows in rising and falling order, in plateaus, with the largest values in one vector, at the ends, or all equal."""
    from mgwfbp_b200.ops.logprob import token_log_probs
    for dtype in TYPES:
        for v in (50261, 10000, 700):
            base = torch.linspace(-4, 9, v, device='cuda')
            kinds = [base, base.flip(0), (base * 3).round() / 3, torch.zeros(v, device='cuda'), base * 0 - 1e4, base.clone()]
            kinds[4][v - 3:] = 5.0
            kinds[4][:2] = 5.0
            kinds[5][v // 2:v // 2 + 24] = 11.0
            z = torch.stack([kinds[i % len(kinds)] for i in range(rows)]).to(dtype)
            t = torch.zeros(rows, dtype=torch.int64, device='cuda')
            for top in (1, 20, 32):
                r = token_log_probs(z, t, top=top)
                lp, bound, order = Rows(z, t).top(top)
                assert torch.equal(r.top_tokens, order)
                assert_within(r.top_logprob, lp, bound, 'top')


def test_log_probs_shapes_and_strides():
    from mgwfbp_b200.ops.logprob import token_log_probs
    z = torch.randn(4, 5, 64, device='cuda')
    t = torch.randint(0, 64, (4, 5), device='cuda')
    r = token_log_probs(z, t, top=3)
    assert r.logprob.shape == r.entropy.shape == (4, 5) and r.top_tokens.shape == r.top_logprob.shape == (4, 5, 3)
    want = Rows(z, t)
    assert_within(r.logprob.reshape(-1), *want.logprob(), 'batched')
    zt = z.transpose(0, 1).detach().requires_grad_()                             # rows in another order
    q = token_log_probs(zt, t.t(), top=3)
    assert torch.equal(q.logprob, r.logprob.t()) and torch.equal(q.top_tokens, r.top_tokens.transpose(0, 1))
    (dz,) = torch.autograd.grad(q.logprob.sum(), zt)
    assert dz.shape == zt.shape
    cols = torch.randn(64, 7, device='cuda').t()                                 # columns of another matrix
    c = token_log_probs(cols, t.reshape(-1)[:7])
    assert torch.equal(c.logprob, token_log_probs(cols.contiguous(), t.reshape(-1)[:7]).logprob)
    e = token_log_probs(torch.randn(1, 64, device='cuda').expand(6, 64), torch.zeros(6, dtype=torch.int64, device='cuda'))
    assert (e.logprob == e.logprob[0]).all()
    none = token_log_probs(z[:0], t[:0], top=2)
    assert none.logprob.shape == (0, 5) and none.top_tokens.shape == (0, 5, 2)


def test_log_probs_offsets_beyond_32_bits():
    from mgwfbp_b200.ops.logprob import token_log_probs
    ld = 1_200_000_000
    store = torch.empty(2 * ld + 1000, dtype=torch.bfloat16, device='cuda')
    z = store.as_strided((3, 1000), (ld, 1))
    z.copy_(torch.randn(3, 1000, device='cuda'))
    t = torch.tensor([1, 2, 3], device='cuda')
    want = Rows(z, t)
    r = token_log_probs(z.detach().requires_grad_(), t, top=4)
    assert_within(r.logprob, *want.logprob(), 'logprob')
    assert torch.equal(r.top_tokens, want.top(4)[2])
    zz = z.detach().requires_grad_()
    (dz,) = torch.autograd.grad(token_log_probs(zz, t).logprob.sum(), zz)
    assert dz.is_contiguous()                                                    # not as far apart as the logits
    one = torch.ones(3, device='cuda')
    assert_within(dz, *want.grad(one, one * 0, torch.bfloat16), 'dz')


# ------------------------------------------------------------------------------------------------------------- clipping
def _grads(sizes, dtypes, gen, sd=1.0, offset=0):
    """Tensors one behind the other in one buffer per type, so that their addresses have every alignment."""
    out = []
    for dt in dtypes:
        mine = [n for i, n in enumerate(sizes) if dtypes[i % len(dtypes)] == dt]
        flat = (torch.randn(sum(mine) + offset, device='cuda', generator=gen) * sd).to(dt)
        at = offset
        for n in mine:
            out.append(flat[at:at + n])
            at += n
    return out


def _exact_clip(grads, max_norm, norm_type, scale):
    each = torch.cat([g.double().reshape(-1) for g in grads]) * scale
    norm = torch.linalg.vector_norm(each, norm_type)
    c = torch.clamp(max_norm / (norm + 1e-6), max=1.0)
    return norm, [g.double() * scale * c for g in grads]


@pytest.mark.parametrize('norm_type', [2.0, 1.0, math.inf])
@pytest.mark.parametrize('sizes,dtypes,offset', [
    ([1], [torch.float32], 0), ([1, 2, 3, 5, 7], [torch.bfloat16], 1), ([5], [torch.float16], 3), ([0, 8192, 0, 8193, 8191], [torch.float32], 1),
    ([100003, 17, 16384 * 3 + 5, 4], TYPES, 5), ([7] * 130, [torch.bfloat16, torch.float32], 0), ([33] * 1100, [torch.float16], 0),
    ([3_000_001, 5_000_003], [torch.bfloat16], 0), ([20_000_000], [torch.float32], 2)])
def test_clip_and_norm(sizes, dtypes, offset, norm_type):
    from mgwfbp_b200.ops.clip import clip_grad_norm_, grad_norm
    gen = torch.Generator(device='cuda').manual_seed(len(sizes))
    for scale, limit in ((1.0, 0.3), (2.0, 0.01), (0.125, 1e30)):
        grads = _grads(sizes, dtypes, gen, offset=offset)
        want_norm, want = _exact_clip(grads, limit, norm_type, scale)
        params = [torch.nn.Parameter(torch.empty_like(g)) for g in grads]
        for p, g in zip(params, grads):
            p.grad = g
        before = grad_norm(grads, norm_type, scale)
        norm = clip_grad_norm_(params, limit, norm_type, grad_scale=scale)
        # a thread's sum of at most 32 values is off by 32 U relatively (positive terms, one rounding each), their 64-bit
        # total by no more, its root by half of that; then one rounding to fp32
        assert_within(norm, want_norm, want_norm * U * (33.01 if norm_type == 1.0 else 17.01), 'norm')
        assert torch.equal(norm, before)
        for g, w in zip(grads, want):                          # the norm, the factor and the product in fp32, the result in the type
            assert_within(g, w, w.abs() * (half_step(g.dtype) + (34.1 if norm_type == 1.0 else 18.1) * U) + tiny(g.dtype), 'grad')


def test_clip_leaves_small_gradients_alone():
    from mgwfbp_b200.ops.clip import clip_grad_norm_
    p = torch.nn.Parameter(torch.zeros(1000, device='cuda'))
    p.grad = torch.randn(1000, device='cuda')
    keep = p.grad.clone()
    clip_grad_norm_([p], 1e6)
    assert torch.equal(p.grad, keep)


def test_clip_values_whose_squares_leave_fp32():
    from mgwfbp_b200.ops.clip import clip_grad_norm_
    for v in (1e-30, 1e30, 3e38, 1e-42):
        p = torch.nn.Parameter(torch.zeros(64, device='cuda'))
        p.grad = torch.full((64,), v, device='cuda')
        x = float(p.grad[0])
        norm = clip_grad_norm_(p, 1.0)
        want = 8.0 * x
        if want <= torch.finfo(torch.float32).max:
            assert abs(float(norm) - want) <= want * U * 1.01 + tiny(torch.float32)
        else:
            assert math.isinf(float(norm))
        w = torch.full((64,), x * min(1.0, 1.0 / (want + 1e-6)), dtype=torch.float64)
        assert_within(p.grad, w, w * 3.1 * U + 2 * tiny(torch.float32), 'grad')


@pytest.mark.parametrize('value', [math.nan, math.inf])
@pytest.mark.parametrize('norm_type', [2.0, 1.0, math.inf])
def test_clip_nonfinite_is_the_librarys(value, norm_type):
    from mgwfbp_b200.ops.clip import clip_grad_norm_
    mine = [torch.nn.Parameter(torch.zeros(n, device='cuda')) for n in (5, 70000)]
    theirs = [torch.nn.Parameter(torch.zeros(n, device='cuda')) for n in (5, 70000)]
    for p, q in zip(mine, theirs):
        p.grad = torch.randn_like(p)
        q.grad = p.grad.clone()
    for ps in (mine, theirs):
        ps[1].grad[69999] = value
    keep = mine[0].grad.clone()
    with pytest.raises(RuntimeError, match='non-finite'):
        clip_grad_norm_(mine, 1.0, norm_type, error_if_nonfinite=True)
    assert torch.equal(mine[0].grad, keep)
    a, b = clip_grad_norm_(mine, 1.0, norm_type), torch.nn.utils.clip_grad_norm_(theirs, 1.0, norm_type)
    assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.isinf(), b.isinf())
    for p, q in zip(mine, theirs):
        torch.testing.assert_close(p.grad, q.grad, equal_nan=True)


def test_clip_layouts_repeats_and_overlaps():
    from mgwfbp_b200.ops.clip import clip_grad_norm_
    p = torch.nn.Parameter(torch.zeros(4, 3, 5, 5, device='cuda').contiguous(memory_format=torch.channels_last))
    p.grad = torch.randn(4, 3, 5, 5, device='cuda').contiguous(memory_format=torch.channels_last)
    q = torch.nn.Parameter(torch.zeros(8, 6, device='cuda').t())
    q.grad = torch.randn(8, 6, device='cuda').t()
    want_norm, want = _exact_clip([p.grad, q.grad], 0.5, 2.0, 1.0)
    norm = clip_grad_norm_([p, q, p, q], 0.5)                                    # each counts and is scaled once
    assert_within(norm, want_norm, want_norm * U * 17.01, 'norm')
    for g, w in zip((p.grad, q.grad), want):
        assert_within(g, w, w.abs() * 19.1 * U, 'grad')
    flat = torch.randn(100, device='cuda')
    a, b = torch.nn.Parameter(torch.zeros(60, device='cuda')), torch.nn.Parameter(torch.zeros(60, device='cuda'))
    a.grad, b.grad = flat[:60], flat[40:]
    keep = flat.clone()
    with pytest.raises(ValueError, match='share memory'):
        clip_grad_norm_([a, b], 0.1)
    assert torch.equal(flat, keep)
    a.grad = torch.randn(1, device='cuda').expand(60)
    with pytest.raises(ValueError, match='stretch of memory'):
        clip_grad_norm_([a], 0.1)
    a.grad, b.grad = flat[:60].clone(), None
    c = torch.nn.Parameter(torch.zeros(3))
    c.grad = torch.zeros(3)
    with pytest.raises(ValueError, match='one device'):
        clip_grad_norm_([a, c], 0.1)


def test_clip_offsets_beyond_32_bits():
    from mgwfbp_b200.ops.clip import clip_grad_norm_
    n = (1 << 32) + 12345
    p = torch.nn.Parameter(torch.empty(0, dtype=torch.bfloat16, device='cuda'))
    g = torch.zeros(n, dtype=torch.bfloat16, device='cuda')
    g[-1], g[(1 << 32) - 1], g[0] = 3.0, 4.0, 12.0
    p.data = g                                                                   # a gradient needs its parameter's shape
    p.grad = g
    norm = clip_grad_norm_(p, 6.5)
    assert float(norm) == 13.0
    assert float(g[-1]) == 1.5 and float(g[(1 << 32) - 1]) == 2.0 and float(g[0]) == 6.0


# -------------------------------------------------------------------------------------------- streams, graphs, together
def _together(net, tokens, targets):
    """One training step's operators as a language model calls them."""
    from mgwfbp_b200.ops.clip import clip_grad_norm_
    from mgwfbp_b200.ops.embedding import embedding
    from mgwfbp_b200.ops.logprob import cross_entropy, token_log_probs
    table, out = net
    x = embedding(tokens, table, scale=2.0, padding_idx=0)
    z = x.reshape(-1, x.shape[-1]) @ out
    loss = cross_entropy(z, targets.reshape(-1), ignore_index=0)
    dt, do = torch.autograd.grad(loss, [table, out])
    table.grad, out.grad = dt, do
    norm = clip_grad_norm_([table, out], 0.05)
    r = token_log_probs(z.detach(), targets.reshape(-1), top=3, ignore_index=0)
    return [loss.detach(), norm, dt, do, r.logprob, r.entropy, r.top_logprob, r.top_tokens]


def _together_inputs(seed, n=300):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    tokens = torch.randint(0, 501, (n,), device='cuda', generator=gen)
    tokens[::7] = 0
    return tokens, torch.roll(tokens, -1)


def _together_net():
    gen = torch.Generator(device='cuda').manual_seed(1)
    table = (torch.randn(501, 64, device='cuda', generator=gen) * 0.1).requires_grad_()
    return table, (torch.randn(64, 501, device='cuda', generator=gen) * 0.1).requires_grad_()


def test_operators_together_match_64_bits():
    net, (tokens, targets) = _together_net(), _together_inputs(2)
    prev = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    try:
        loss, norm, dt, do, logprob, entropy, tlp, tt = _together(net, tokens, targets)
    finally:
        torch.backends.cuda.matmul.allow_tf32 = prev
    table, out = (p.detach().double().requires_grad_() for p in net)
    x = torch.nn.functional.embedding(tokens, table, padding_idx=0) * 2.0
    z = x @ out
    want = torch.nn.functional.cross_entropy(z, targets, ignore_index=0)
    want.backward()
    total = torch.nn.utils.clip_grad_norm_([table, out], 0.05)
    torch.testing.assert_close(loss.double(), want.detach(), rtol=1e-5, atol=1e-6)
    torch.testing.assert_close(norm.double(), total, rtol=1e-5, atol=1e-6)
    torch.testing.assert_close(dt.double(), table.grad, rtol=1e-4, atol=1e-6)
    torch.testing.assert_close(do.double(), out.grad, rtol=1e-4, atol=1e-6)
    keep = targets != 0
    lp = torch.log_softmax(z.detach(), 1)
    torch.testing.assert_close(logprob[keep].double(), lp[keep].gather(1, targets[keep, None]).squeeze(1), rtol=1e-5, atol=1e-5)
    assert not logprob[~keep].any() and (tt[~keep] == -1).all()


def test_operators_on_another_stream_and_in_two_graphs():
    """Two captured graphs replayed in turn and on streams of their own give what eager calls give, bit for bit."""
    net = _together_net()
    sets = [_together_inputs(s) for s in (5, 6)]
    want = [[v.clone() for v in _together(net, *s)] for s in sets]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = _together(net, *sets[1])
    side.synchronize()
    for a, b in zip(got, want[1]):
        assert torch.equal(a, b)
    graphs, outs, statics = [], [], []
    for s in sets:
        static = [v.clone() for v in s]
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = _together(net, *static)
        graphs.append(g)
        outs.append(o)
        statics.append(static)
    for turn in range(3):                                      # the graphs' inputs change places
        for k in (0, 1):
            for st, v in zip(statics[k], sets[(k + turn) % 2]):
                st.copy_(v)
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        torch.cuda.synchronize()
        for k in (0, 1):                                       # both at once
            with torch.cuda.stream(streams[k]):
                graphs[k].replay()
        torch.cuda.synchronize()
        for k in (0, 1):
            for a, b in zip(outs[k], want[(k + turn) % 2]):
                assert torch.equal(a, b)
    from mgwfbp_b200.ops.embedding import check_status
    check_status()


def test_first_call_inside_a_capture():
    """A process whose first use of the operators is being captured."""
    import subprocess
    import sys
    code = """
import torch
from test_gpu_lm_ops import _together, _together_inputs, _together_net
net, data = _together_net(), _together_inputs(4)
a = torch.randn(64, 64, device='cuda', requires_grad=True)
torch.autograd.grad((a @ a).sum(), a)                      # the library's own first calls
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    got = _together(net, *data)
g.replay()
torch.cuda.synchronize()
got = [v.clone() for v in got]
want = _together(net, *data)
assert all(torch.equal(x, y) for x, y in zip(got, want))
print('captured')
"""
    import os
    here = os.path.dirname(os.path.abspath(__file__))
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([here, os.path.dirname(here)]))
    out = subprocess.run([sys.executable, '-c', code], capture_output=True, text=True, timeout=300, env=env)
    assert out.returncode == 0 and 'captured' in out.stdout, out.stderr[-2000:]


def test_other_types_run_the_parents():
    from mgwfbp_b200.ops.embedding import FusedEmbedding
    from mgwfbp_b200.ops.logprob import FusedCrossEntropyLoss
    t = torch.tensor([1, 3], device='cuda')
    e = FusedEmbedding(5, 4, scale=2.0).cuda().double()
    assert torch.equal(e(t), e.weight[t] * 2.0)
    z = torch.randn(2, 5, device='cuda', dtype=torch.float64)
    assert torch.equal(FusedCrossEntropyLoss()(z, t), torch.nn.functional.cross_entropy(z, t))


def test_native_launches_are_counted():
    from mgwfbp_b200.ops import counters
    before = counters.snapshot()
    _together(_together_net(), *_together_inputs(3))
    seen = counters.diff(before)
    for name in ('embedding_fwd', 'embedding_grad', 'logprob_fwd', 'grad_norm', 'grad_scale'):
        assert seen.get(name, 0) >= 1, (name, seen)


def test_refusals_on_the_gpu():
    from mgwfbp_b200.ops.clip import grad_norm
    from mgwfbp_b200.ops.embedding import embedding, embedding_grad
    from mgwfbp_b200.ops.logprob import token_log_probs
    w, t = torch.randn(5, 4, device='cuda', dtype=torch.float64), torch.tensor([1], device='cuda')
    with pytest.raises(TypeError, match='float32, float16 or bfloat16'):
        embedding(t, w)
    with pytest.raises(TypeError, match='float32, float16 or bfloat16'):
        embedding_grad(w[:1], t, 5)
    with pytest.raises(TypeError, match='float32, float16 or bfloat16'):
        token_log_probs(w[:1], t)
    with pytest.raises(TypeError, match='float32, float16 or bfloat16'):
        grad_norm([w])
    with pytest.raises(ValueError, match='tokens are on'):
        embedding(t.cpu(), w.float())
    with pytest.raises(ValueError, match='tokens are on'):
        token_log_probs(w[:1].float(), t.cpu())
    with pytest.raises(RuntimeError):                          # differentiable once
        x = w.float().requires_grad_()
        (g,) = torch.autograd.grad(token_log_probs(x[:1], t).logprob.sum(), x, create_graph=True)
        torch.autograd.grad(g.sum(), x)


@pytest.mark.parametrize('kind', ['embedding', 'log_probs', 'cross_entropy'])
def test_gradients_are_differentiable_once(kind):
    """A second derivative raises an error, also where the incoming gradient has no graph of its own."""
    from mgwfbp_b200.ops.embedding import embedding
    from mgwfbp_b200.ops.logprob import cross_entropy, token_log_probs
    t = torch.tensor([1, 3, 3], device='cuda')
    w = torch.randn(5, 4, device='cuda', requires_grad=True)
    z = torch.randn(3, 7, device='cuda', requires_grad=True)
    if kind == 'embedding':
        up = torch.randn(3, 4, device='cuda', requires_grad=True)
        leaf, out = w, (embedding(t, w) * up).sum()
    else:
        leaf, out = z, token_log_probs(z, t).logprob.sum() if kind == 'log_probs' else cross_entropy(z, t)
    (plain,) = torch.autograd.grad(out, leaf, retain_graph=True)
    assert not plain.requires_grad
    (g,) = torch.autograd.grad(out, leaf, create_graph=True)
    assert torch.equal(g, plain) and g.requires_grad
    with pytest.raises(RuntimeError, match='differentiate twice'):
        (g.square().sum() + out).backward()


def test_graph_is_released_and_guards_its_inputs():
    """Nothing outlives the graph, a released graph is refused, and so are inputs that changed since."""
    import gc
    from mgwfbp_b200.ops.embedding import embedding
    from mgwfbp_b200.ops.logprob import cross_entropy, token_log_probs
    t = torch.randint(0, 1000, (512,), device='cuda')
    w = torch.randn(1000, 256, device='cuda', requires_grad=True)
    z = torch.randn(512, 1000, device='cuda', requires_grad=True)

    def forward():
        return [embedding(t, w), token_log_probs(z, t, top=3).logprob, token_log_probs(z, t).entropy, cross_entropy(z, t)]
    for out in forward():                                      # the first calls' own memory
        out.sum().backward()
    w.grad = z.grad = out = None
    gc.collect()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    for turn in range(2):
        for out in forward():
            if turn:
                total = out.sum()
                total.backward()
                with pytest.raises(RuntimeError, match='second time'):
                    total.backward()
                total = None
        w.grad = z.grad = out = None                           # (with turn 0: graphs that never ran backward)
        torch.cuda.synchronize()
        assert torch.cuda.memory_allocated() == before
    for k in (1, 2, 3):
        out = forward()[k]
        with torch.no_grad():
            z.mul_(1.0)
        with pytest.raises(RuntimeError, match='modified by an inplace operation'):
            out.sum().backward()
    out = forward()[0]
    t.add_(0)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        out.sum().backward()


def test_clip_marks_gradients_as_changed():
    from mgwfbp_b200.ops.clip import clip_grad_norm_
    p = torch.nn.Parameter(torch.zeros(8, device='cuda'))
    p.grad = torch.ones(8, device='cuda')
    x = torch.ones(8, device='cuda', requires_grad=True)
    y = (x * p.grad).sum()                                     # saves the gradient
    clip_grad_norm_([p], 0.5)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.backward()


def test_clip_with_parameters_on_the_host_that_have_no_gradient():
    from mgwfbp_b200.ops.clip import clip_grad_norm_
    from mgwfbp_b200.ops import counters
    ps = [torch.nn.Parameter(torch.zeros(3)), torch.nn.Parameter(torch.zeros(3, device='cuda'))]
    ps[1].grad = torch.full((3,), 2.0, device='cuda')
    before = counters.snapshot()
    clip_grad_norm_(iter(ps), 1.0)
    assert counters.diff(before) == {'grad_norm': 1, 'grad_scale': 1}
    assert abs(ps[1].grad.norm().item() - 1.0) < 1e-5          # max_norm / (norm + 1e-6): 3e-7 below 1


@pytest.mark.parametrize('n,dim', [(5000, 131), (1024, 16500), (1025, 16500), (40000, 451), (65536, 260), (65537, 260)])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_embedding_sorted_beside_the_lookup(n, dim, dtype):
    """The gradient through the graph, whose tokens the lookup's launch has sorted, is the gradient of the plain call bit for bit,
    whatever runs before and behind it in the stream, also twice and with padding and tokens outside."""
    from mgwfbp_b200.ops.embedding import check_status, embedding, embedding_grad
    from mgwfbp_b200.ops._tokens import TokenIndexError
    gen = torch.Generator(device='cuda').manual_seed(n)
    vocab = 777
    w = torch.randn(vocab, dim, device='cuda', generator=gen).to(dtype).requires_grad_()
    dy = torch.randn(n, dim, device='cuda', generator=gen).to(dtype)
    for turn in range(4):
        t = torch.randint(0, vocab, (n,), device='cuda', generator=gen)
        out = embedding(t, w, 0.5, 3)
        assert torch.equal(out, (w.detach()[t].float() * 0.5).to(dtype))
        order_of_release = [torch.full((n,), 9, dtype=torch.int64, device='cuda') for _ in range(3)]     # memory moves on
        (dw,) = torch.autograd.grad(out, w, dy, retain_graph=True)
        (again,) = torch.autograd.grad(out, w, dy)
        want = embedding_grad(dy, t, vocab, 0.5, 3)
        assert torch.equal(dw, want) and torch.equal(again, want)
        del order_of_release
    t[n // 2] = vocab
    (dw,) = torch.autograd.grad(embedding(t, w, 0.5, 3), w, dy)
    with pytest.raises(TokenIndexError, match='embedding: token 777 at position %d' % (n // 2)):
        check_status()
    want = embedding_grad(dy, t, vocab, 0.5, 3)
    with pytest.raises(TokenIndexError, match='embedding gradient: token 777'):
        check_status()
    assert torch.equal(dw, want)


def test_embedding_sorted_beside_the_lookup_in_a_graph():
    from mgwfbp_b200.ops.embedding import embedding, embedding_grad
    n, vocab, dim = 20000, 3001, 510
    w = torch.randn(vocab, dim, device='cuda', requires_grad=True)
    t = torch.randint(0, vocab, (n,), device='cuda')
    dy = torch.randn(n, dim, device='cuda')
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.autograd.grad(embedding(t, w), w, dy)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = embedding(t, w)
        (dw,) = torch.autograd.grad(out, w, dy)
    for seed in range(5):
        t.copy_(torch.randint(0, vocab, (n,), device='cuda', generator=torch.Generator(device='cuda').manual_seed(seed)))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, w.detach()[t]) and torch.equal(dw, embedding_grad(dy, t, vocab))


def test_two_threads_on_two_streams():
    """The host side runs without the interpreter's lock: two threads at once, each on its own stream."""
    import threading
    from mgwfbp_b200.ops.clip import clip_grad_norm_
    from mgwfbp_b200.ops.embedding import check_status, embedding
    from mgwfbp_b200.ops.logprob import cross_entropy, token_log_probs

    def inputs(seed):
        gen = torch.Generator(device='cuda').manual_seed(seed)
        w = torch.randn(3001, 512, device='cuda', generator=gen, requires_grad=True)
        z = torch.randn(300, 5003, device='cuda', generator=gen, requires_grad=True)
        return (torch.randint(0, 3001, (17000,), device='cuda', generator=gen), w, torch.randn(17000, 512, device='cuda', generator=gen), z,
                torch.randint(0, 5003, (300,), device='cuda', generator=gen))

    def once(t, w, dy, z, chosen):
        out = embedding(t, w, 2.0)
        (dw,) = torch.autograd.grad(out, w, dy)
        r = token_log_probs(z, chosen, top=7)
        (dz,) = torch.autograd.grad(r.logprob.sum() + r.entropy.sum(), z)
        loss = cross_entropy(z, chosen)
        (dl,) = torch.autograd.grad(loss, z)
        p = torch.nn.Parameter(torch.zeros_like(dw))
        p.grad = dw.clone()
        norm = clip_grad_norm_([p], 1.0)
        return [out.detach(), dw, r.logprob.detach(), r.entropy.detach(), r.top_logprob, r.top_tokens, dz, loss.detach(), dl, norm, p.grad]
    data = [inputs(k) for k in range(2)]
    want = [once(*d) for d in data]
    torch.cuda.synchronize()
    faults = []

    def work(k):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(15):
                    got = once(*data[k])
                    stream.synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[k])):
                        faults.append('thread %d: other values' % k)
        except Exception as e:                                 # a thread's exception would be lost
            faults.append('thread %d: %r' % (k, e))
    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join(120)
        assert not th.is_alive()
    assert not faults, faults
    check_status()


def test_native_errors_carry_their_text():
    """What the library refuses comes back as the package's error, from the caller's thread and from the backward pass."""
    import ctypes as C
    from mgwfbp_b200.ops import _lib, _tokens, counters
    m, lib = _tokens.native(), _lib.load(allow_build=False)
    t, w = torch.tensor([0, 1], device='cuda'), torch.zeros(3, 4, device='cuda', requires_grad=True)
    z = torch.zeros(2, 4, device='cuda', requires_grad=True)
    out, loss = m.embedding(t, w, 1.0, -1), m.cross_entropy(z, t, -100, True, 1.0)
    before = counters.snapshot()
    with pytest.raises(ValueError, match='share memory'):
        m.clip_grads([w.detach()[:2].view(-1), w.detach()[1:].view(-1)], False, 0, 1.0, 1.0, True)
    real = {name: C.cast(getattr(lib, name), C.c_void_p).value for name in _tokens._FUNCTIONS}
    failing = C.CFUNCTYPE(C.c_int)(lambda: 7)                  # stands in for every launch: nothing reaches the GPU
    fake = {k: v if k == 'mgw_last_error' or k.endswith('_bytes') else C.cast(failing, C.c_void_p).value for k, v in real.items()}
    m.bind(fake, _tokens.status_words(), _lib.NativeLibraryError)
    try:
        for what, call in (('embedding_fwd', lambda: m.embedding(t, w, 1.0, -1)), ('embedding_grad', lambda: m.embedding_grad(z, t, 3, 1.0, -1)),
                           ('logprob_fwd', lambda: m.token_log_probs(z, t, -100, 1)),
                           ('cross_entropy_fwd', lambda: m.cross_entropy(z, t, -100, True, 1.0)),
                           ('grad_clip', lambda: m.clip_grads([z.detach()], False, 0, 1.0, 1.0, True))):
            with pytest.raises(_lib.NativeLibraryError, match='%s failed with code 7' % what):
                call()
        for what, x in (('embedding_grad', out.sum()), ('cross_entropy_bwd', loss)):
            with pytest.raises(RuntimeError, match='%s failed with code 7' % what):
                x.backward()
    finally:
        m.bind(real, _tokens.status_words(), _lib.NativeLibraryError)
    assert counters.diff(before) == {}
    assert torch.equal(m.embedding(t, w, 1.0, -1), w[t])


def test_native_calls_leave_other_arguments_alone():
    """No result, and no launch, for what the kernels do not take: the functions in front say why."""
    from mgwfbp_b200.ops import counters
    from mgwfbp_b200.ops._tokens import native
    m, t, w = native(), torch.tensor([0, 1], device='cuda'), torch.zeros(3, 4, device='cuda')
    before = counters.snapshot()
    for got in (m.embedding(t.cpu(), w, 1.0, -1), m.embedding(t, w.double(), 1.0, -1), m.embedding(t, w[0], 1.0, -1),
                m.embedding(t.float(), w, 1.0, -1), m.embedding(t, w[:0], 1.0, -1), m.embedding(t, w[:, :0], 1.0, -1),
                m.embedding_grad(w[:2], t, 0, 1.0, -1), m.embedding_grad(w, t, 3, 1.0, -1), m.token_log_probs(w, t, -100, 1),
                m.token_log_probs(w[:2], t, -100, 5), m.token_log_probs(w[:2], t, -100, -1), m.token_log_probs(w[:2], t[:, None], -100, 1),
                m.cross_entropy(w, t, -100, True, 1.0), m.cross_entropy(w[:2].double(), t, -100, True, 1.0),
                m.clip_grads([w.double()], False, 0, 1.0, 1.0, True), m.clip_grads([w[:, ::2]], False, 0, 1.0, 1.0, True),
                m.clip_grads([w, w.cpu()], False, 0, 1.0, 1.0, True), m.clip_grads([], False, 0, 1.0, 1.0, True)):
        assert got is None
    assert counters.diff(before) == {}


@pytest.mark.parametrize('n', [700, 20000, 70000])
@pytest.mark.parametrize('before', ['copy', 'fill', 'join', 'nothing'])
def test_captured_behind_other_nodes(n, before):
    """In a captured graph the launches may follow a copy, a fill, two branches or nothing, not only a kernel."""
    from mgwfbp_b200.ops.embedding import embedding, embedding_grad
    vocab, dim = 3001, 500
    w = torch.randn(vocab, dim, device='cuda', requires_grad=True)
    t, dy = torch.zeros(n, dtype=torch.int64, device='cuda'), torch.randn(n, dim, device='cuda')
    source, other = torch.randint(0, vocab, (n,), device='cuda'), torch.zeros(4, device='cuda')
    side = torch.cuda.Stream()

    def call():
        main = torch.cuda.current_stream()
        if before == 'copy':
            t.copy_(source)
        elif before == 'fill':
            other.zero_()
        elif before == 'join':
            side.wait_stream(main)
            with torch.cuda.stream(side):
                other.add_(1)
            t.copy_(source)
            main.wait_stream(side)
        a = embedding_grad(dy, t, vocab)
        out = embedding(t, w)
        (b,) = torch.autograd.grad(out, w, dy)
        return a, out, b
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = call()
    for _ in range(3):
        source.copy_(torch.randint(0, vocab, (n,), device='cuda'))
        if before in ('fill', 'nothing'):
            t.copy_(source)
        g.replay()
        torch.cuda.synchronize()
        want = embedding_grad(dy, source, vocab)
        assert torch.equal(got[0], want) and torch.equal(got[2], want) and torch.equal(got[1], w.detach()[source])


@pytest.mark.parametrize('how', ['offload', 'checkpoint', 'anomaly', 'hooks'])
def test_graph_features(how):
    """Saved tensors that are moved away or computed again, anomaly mode and hooks on tensors: the same gradients."""
    from torch.utils.checkpoint import checkpoint
    from mgwfbp_b200.ops.embedding import embedding
    from mgwfbp_b200.ops.logprob import cross_entropy, token_log_probs
    w = torch.randn(777, 96, device='cuda', requires_grad=True)
    head = torch.randn(1003, 96, device='cuda', requires_grad=True)
    t, chosen = torch.randint(0, 777, (2000,), device='cuda'), torch.randint(0, 1003, (2000,), device='cuda')

    def model(table, out):
        z = embedding(t, table, 0.1) @ out.t()
        r = token_log_probs(z, chosen, top=2)
        return cross_entropy(z, chosen) + 0.01 * r.entropy.mean() - r.logprob.mean()
    want = torch.autograd.grad(model(w, head), (w, head))
    if how == 'offload':
        with torch.autograd.graph.save_on_cpu():
            loss = model(w, head)
        got = torch.autograd.grad(loss, (w, head))
    elif how == 'checkpoint':
        got = torch.autograd.grad(checkpoint(model, w, head, use_reentrant=False), (w, head))
    elif how == 'anomaly':
        with torch.autograd.set_detect_anomaly(True):
            got = torch.autograd.grad(model(w, head), (w, head))
    else:
        seen = []
        rows = embedding(t, w, 0.1)
        rows.register_hook(lambda g: seen.append(g.shape))
        z = rows @ head.t()
        z.retain_grad()
        r = token_log_probs(z, chosen, top=2)
        loss = cross_entropy(z, chosen)
        loss.register_hook(lambda g: g * 1.0)
        got = torch.autograd.grad(loss + 0.01 * r.entropy.mean() - r.logprob.mean(), (w, head))
        assert seen == [rows.shape]
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.inference_mode():
        assert torch.equal(model(w, head), model(w.detach(), head.detach())) and not model(w, head).requires_grad
    with torch.no_grad():
        assert not embedding(t, w).requires_grad and embedding(t, w).grad_fn is None
