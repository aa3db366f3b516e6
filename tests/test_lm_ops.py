"""Embedding, token log probabilities, cross entropy and gradient clipping without a GPU: what the functions compute on
CPU tensors, what they refuse, and the refusals of the native entry points."""
import ctypes as C
import math

import pytest
import torch

from lm_oracle import Rows, assert_within, embedding_grad as oracle_grad, half_step, tiny
from mgwfbp_b200.ops import _lib, clip, embedding as emb, logprob as lp


# ---------------------------------------------------------------------------------------------------------- embedding
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('scale,padding', [(1.0, None), (2.5, 3), (-0.5, -1)])
def test_embedding_and_gradient_on_cpu(dtype, scale, padding):
    torch.manual_seed(0)
    w = torch.randn(11, 5).to(dtype).requires_grad_()
    t = torch.tensor([[1, 3, 3, 10], [0, 10, 10, 3]])
    out = emb.embedding(t, w, scale, padding)
    assert_within(out, w.detach().double()[t] * scale, half_step(dtype) * out.detach().double().abs() + tiny(dtype), 'out')
    dy = torch.randn(2, 4, 5).to(dtype)
    (dw,) = torch.autograd.grad(out, w, dy)
    want, bound = oracle_grad(dy, t, 11, scale, None if padding is None else padding % 11)
    assert_within(dw, want, bound, 'dw')


def test_embedding_gradient_against_differences():
    w = torch.randn(6, 3, dtype=torch.float64, requires_grad=True)
    t = torch.tensor([0, 5, 5, 2])
    assert torch.autograd.gradcheck(lambda x: emb.embedding(t, x, 1.5), (w,))


def test_embedding_without_tokens():
    w = torch.randn(4, 3, requires_grad=True)
    t = torch.empty(2, 0, dtype=torch.int64)
    out = emb.embedding(t, w)
    assert out.shape == (2, 0, 3)
    assert torch.equal(emb.embedding_grad(torch.empty(2, 0, 3), t, 4), torch.zeros(4, 3))


def test_embedding_refusals():
    w = torch.randn(4, 3)
    t = torch.tensor([1, 2])
    with pytest.raises(TypeError, match='int32 or int64'):
        emb.embedding(t.float(), w)
    with pytest.raises(ValueError, match='non-empty'):
        emb.embedding(t, torch.randn(4))
    with pytest.raises(ValueError, match='non-empty'):
        emb.embedding(t, torch.randn(4, 0))
    with pytest.raises(ValueError, match='padding_idx'):
        emb.embedding(t, w, padding_idx=4)
    with pytest.raises(IndexError):
        emb.embedding(torch.tensor([4]), w)
    with pytest.raises(ValueError, match='shape of tokens'):
        emb.embedding_grad(torch.randn(3, 3), t, 4)
    with pytest.raises(ValueError, match='positive'):
        emb.embedding_grad(torch.randn(2, 3), t, 0)
    for option in ({'max_norm': 1.0}, {'sparse': True}, {'scale_grad_by_freq': True}):
        with pytest.raises(ValueError, match='does not support'):
            emb.FusedEmbedding(4, 3, **option)


def test_fused_embedding_is_an_embedding():
    torch.manual_seed(3)
    a = emb.FusedEmbedding(9, 4, padding_idx=2)
    torch.manual_seed(3)
    b = torch.nn.Embedding(9, 4, padding_idx=2)
    assert list(a.state_dict()) == list(b.state_dict())
    t = torch.tensor([[1, 2], [8, 8]])
    assert torch.equal(a(t), b(t))
    a(t).sum().backward()
    b(t).sum().backward()
    assert torch.equal(a.weight.grad, b.weight.grad)


# ----------------------------------------------------------------------------------------------------- log probabilities
def _logits(rows=6, vocab=37, seed=0):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(rows, vocab, generator=g) * 3
    z[1, 5:] = -math.inf                                   # five tokens are left
    z[2, 7] = torch.finfo(torch.float32).min
    z[3, :] = 2.0                                          # all equal
    t = torch.randint(0, 5, (rows,), generator=g)
    t[4] = -100
    return z, t


def test_log_probs_on_cpu():
    z, t = _logits()
    z[4] = math.nan                                        # padding: never read
    r = lp.token_log_probs(z, t, top=4)
    want = Rows(z, t)
    assert_within(r.logprob, *want.logprob(), 'logprob')
    assert_within(r.entropy, *want.entropy(), 'entropy')
    v, bound, order = want.top(4)
    assert torch.equal(r.top_tokens, order)
    assert_within(r.top_logprob, v, bound, 'top')
    assert r.top_tokens[3].tolist() == [0, 1, 2, 3] and r.top_tokens[4].tolist() == [-1] * 4


def test_log_probs_gradient_against_differences():
    z = torch.randn(3, 6, dtype=torch.float64, requires_grad=True)
    t = torch.tensor([0, -100, 5])
    assert torch.autograd.gradcheck(lambda x: lp.token_log_probs(x, t)[:2], (z,))
    assert torch.autograd.gradcheck(lambda x: lp.cross_entropy(x, t), (z,))


def test_oracle_gradient_is_the_formulas_gradient():
    """The 64-bit gradient that the kernels are held to, against automatic differentiation."""
    z, t = _logits(5, 9)
    zd = z.double().requires_grad_()
    g1, g2 = torch.randn(5, dtype=torch.float64), torch.randn(5, dtype=torch.float64)
    r = lp.token_log_probs(zd, t)
    (want,) = torch.autograd.grad((r.logprob * g1 + r.entropy * g2)[t >= 0].sum(), zd)
    got, _ = Rows(z, t).grad(g1, g2, torch.float64)
    torch.testing.assert_close(got, want, rtol=1e-12, atol=1e-14)


@pytest.mark.parametrize('reduction', ['mean', 'sum', 'none'])
def test_cross_entropy_is_the_librarys_on_cpu(reduction):
    z, t = _logits()
    a = torch.nn.functional.cross_entropy(z, t, reduction=reduction)
    b = lp.FusedCrossEntropyLoss(reduction=reduction)(z, t)
    torch.testing.assert_close(a, b, rtol=1e-6, atol=1e-6)
    assert math.isnan(float(lp.cross_entropy(z, torch.full((6,), -100))))


def test_log_prob_refusals():
    z, t = _logits()
    with pytest.raises(TypeError, match='int32 or int64'):
        lp.token_log_probs(z, t.double())
    with pytest.raises(ValueError, match='shape of tokens'):
        lp.token_log_probs(z, t[:5])
    with pytest.raises(ValueError, match='top'):
        lp.token_log_probs(z, t, top=33)
    with pytest.raises(ValueError, match='top'):
        lp.token_log_probs(z[:, :3], t.clamp(max=2), top=4)
    with pytest.raises(TypeError, match='floating'):
        lp.token_log_probs(z.long(), t)
    with pytest.raises(IndexError):
        lp.token_log_probs(z, torch.full((6,), 37))
    with pytest.raises(ValueError, match='reduction'):
        lp.cross_entropy(z, t, reduction='median')
    with pytest.raises(ValueError, match='rows, vocabulary'):
        lp.FusedCrossEntropyLoss()(z.view(2, 3, 37), t.view(2, 3))


# ------------------------------------------------------------------------------------------------------------- clipping
def _params(seed=0, dtypes=(torch.float32, torch.bfloat16, torch.float16)):
    g = torch.Generator().manual_seed(seed)
    out = []
    for i, n in enumerate((1, 7, 64, 1000)):
        p = torch.nn.Parameter(torch.zeros(n).to(dtypes[i % len(dtypes)]))
        p.grad = torch.randn(n, generator=g).to(p.dtype)
        out.append(p)
    out.append(torch.nn.Parameter(torch.zeros(3)))                   # has no gradient
    return out


@pytest.mark.parametrize('norm_type', [1.0, 2.0, math.inf])
def test_clip_is_the_librarys_on_cpu(norm_type):
    mine, theirs = _params(dtypes=(torch.float32,)), _params(dtypes=(torch.float32,))
    a = clip.clip_grad_norm_(mine, 0.7, norm_type)
    b = torch.nn.utils.clip_grad_norm_(theirs, 0.7, norm_type)
    torch.testing.assert_close(a, b, rtol=1e-6, atol=0)
    for p, q in zip(mine[:-1], theirs):
        torch.testing.assert_close(p.grad, q.grad, rtol=1e-6, atol=0)


def test_clip_factor_mixed_types_and_repeats_on_cpu():
    ps = _params()
    before = [p.grad.double() for p in ps[:-1]]
    norm = math.sqrt(sum(float((0.5 * g).square().sum()) for g in before))
    got = clip.clip_grad_norm_(ps + [ps[3]], 1.0, grad_scale=0.5)             # the last one counts once
    assert abs(float(got) - norm) <= 1e-6 * norm
    for p, g in zip(ps, before):
        want = g * 0.5 * min(1.0, 1.0 / (norm + 1e-6))
        assert_within(p.grad, want, half_step(p.dtype) * want.abs() * 1.001 + tiny(p.dtype), 'grad')
    assert float(clip.grad_norm([])) == 0.0 and float(clip.clip_grad_norm_([ps[-1]], 1.0)) == 0.0


def test_clip_refusals():
    ps = _params()
    with pytest.raises(ValueError, match='norm_type'):
        clip.clip_grad_norm_(ps, 1.0, 3.0)
    with pytest.raises(ValueError, match='max_norm'):
        clip.clip_grad_norm_(ps, -1.0)
    with pytest.raises(ValueError, match='max_norm'):
        clip.clip_grad_norm_(ps, math.nan)
    for s in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match='grad_scale'):
            clip.clip_grad_norm_(ps, 1.0, grad_scale=s)
    with pytest.raises(ValueError, match='stretch of memory'):
        clip.grad_norm([torch.randn(4, 6)[:, ::2]])
    with pytest.raises(TypeError, match='dense'):
        clip.grad_norm([torch.zeros(3, dtype=torch.int64)])
    ps[0].grad.fill_(math.nan)
    keep = ps[3].grad.clone()
    with pytest.raises(RuntimeError, match='non-finite'):
        clip.clip_grad_norm_(ps, 1.0, error_if_nonfinite=True)
    assert torch.equal(ps[3].grad, keep)


# ------------------------------------------------------------------------------------------- the native entry points
# Every call below is refused by the host code before anything is launched.
def test_native_embedding_refuses_bad_arguments():
    lib = _lib.load(allow_build=False)
    buf = (C.c_int * 64)()
    p = C.addressof(buf)
    ok = dict(tokens=p, wide=0, n=4, weight=p, ld=4, vocab=8, dim=4, dtype=0, scale=1.0, out=p, order=None,
              padding=-1, status=p, stream=None)
    for bad in (dict(tokens=None), dict(weight=None), dict(out=None), dict(status=None), dict(n=-1), dict(n=1 << 31), dict(vocab=0),
                dict(vocab=(1 << 31) - 1), dict(dim=0), dict(dtype=3), dict(dtype=-1), dict(ld=3), dict(order=p & ~15),
                dict(order=p & ~15, n=65537, dim=1024, ld=1024), dict(order=(p & ~15) + 8, n=2000, dim=8192, ld=8192)):
        assert lib.mgw_embedding_fwd(*{**ok, **bad}.values()) == 2, bad
    for n, there in ((0, False), (1024, False), (1025, True), (65536, True), (65537, False)):
        assert (lib.mgw_embedding_order_bytes(n, 8, 8192, 0) > 0) == there
    assert lib.mgw_embedding_order_bytes(2000, 8, 4195, 0) > 0 == lib.mgw_embedding_order_bytes(2000, 8, 4195, 2)   # 32 MB and 16
    need = lib.mgw_embedding_grad_bytes(2000, 8, 4, 0)             # short lists need no scratch memory
    assert need > 0 and lib.mgw_embedding_grad_bytes(0, 8, 4, 0) == 0 and lib.mgw_embedding_grad_bytes(1024, 8, 4, 0) == 0
    ok = dict(dy=p, ld=4, tokens=p, wide=0, n=2000, vocab=8, dim=4, dtype=0, scale=1.0, padding=-1, order=None, dw=p,
              work=p & ~15, bytes=need, status=p, stream=None)
    for bad in (dict(dy=None), dict(tokens=None), dict(dw=None), dict(work=None), dict(status=None), dict(bytes=need - 1), dict(ld=3),
                dict(work=(p & ~15) + 8), dict(dtype=7), dict(dim=-1), dict(order=p & ~15),
                dict(order=(p & ~15) + 8, dim=8192, ld=8192)):
        assert lib.mgw_embedding_grad(*{**ok, **bad}.values()) == 2, bad


def test_native_logprob_refuses_bad_arguments():
    lib = _lib.load(allow_build=False)
    buf = (C.c_int * 64)()
    p = C.addressof(buf)
    ok = dict(z=p, ld=8, rows=2, vocab=8, dtype=0, tokens=p, wide=0, ignore=-100, logprob=p, entropy=p, stats=p, top=2, tlp=p, tt=p,
              status=p, stream=None)
    for bad in (dict(z=None), dict(tokens=None), dict(logprob=None), dict(status=None), dict(tlp=None), dict(tt=None), dict(top=33),
                dict(top=9), dict(top=-1), dict(vocab=0), dict(ld=7), dict(rows=-1), dict(dtype=5)):
        assert lib.mgw_logprob_fwd(*{**ok, **bad}.values()) == 2, bad
    ok = dict(z=p, ld=8, rows=2, vocab=8, dtype=0, tokens=p, wide=0, ignore=-100, stats=p, entropy=p, g1=p, g2=p, g=None, count=None,
              written=0, expected=1.0, dz=p, dz_ld=8, stream=None)
    for bad in (dict(z=None), dict(stats=None), dict(dz=None), dict(dz_ld=7), dict(entropy=None), dict(g=p), dict(written=1)):
        assert lib.mgw_logprob_bwd(*{**ok, **bad}.values()) == 2, bad
    ok = dict(z=p, ld=8, rows=2, vocab=8, dtype=0, tokens=p, wide=0, ignore=-100, mean=1, expected=1.0, logprob=p, stats=p, loss=p, dz=p,
              dz_ld=8, work=p, status=p, stream=None)
    for bad in (dict(z=None), dict(z=p + 2), dict(tokens=None), dict(logprob=None), dict(loss=None), dict(work=None), dict(status=None),
                dict(dz_ld=7), dict(stats=p + 4), dict(vocab=0), dict(dtype=3)):
        assert lib.mgw_cross_entropy_fwd(*{**ok, **bad}.values()) == 2, bad


def test_native_clip_refuses_bad_arguments():
    lib = _lib.load(allow_build=False)
    buf = (C.c_double * 4096)()
    work, need = C.addressof(buf), lib.mgw_grad_clip_bytes(2)
    assert need <= C.sizeof(buf)

    def call(ptrs=(4096, 8192), numels=(4, 4), dtypes=(0, 0), norm=0, work=work, need=need, out=work):
        n = len(ptrs)
        return lib.mgw_grad_clip((C.c_ulonglong * n)(*ptrs), (C.c_longlong * n)(*numels), bytes(dtypes), n, norm, 1.0, 1.0, 1, work, need,
                                 out, None)
    assert call(norm=3) == 2 and call(work=None) == 2 and call(need=need - 1) == 2 and call(out=None) == 2 and call(work=work + 4) == 2
    assert call(ptrs=(4097, 8192)) == 2 and call(numels=(-1, 4)) == 2 and call(dtypes=(3, 0)) == 2 and call(ptrs=(0, 8192)) == 2
    assert call(ptrs=(4096, 4100)) == 2                                # they share three elements
    assert b'share memory' in lib.mgw_last_error()
    assert call(ptrs=(4096, 4096), numels=(4, 2)) == 2                 # one inside the other
    assert call(ptrs=(4096, 4096), dtypes=(0, 1)) == 2                 # the same place as two types


def test_native_binding_refuses_what_is_not_on_a_gpu():
    """The functions that allocate and launch take CUDA tensors of the kernels' types only, whoever calls them."""
    m = _lib.load_binding()
    t, w = torch.tensor([0, 1]), torch.randn(3, 4)
    for call in (lambda: m.embedding(t, w, 1.0, -1), lambda: m.embedding_grad(w[:2], t, 3, 1.0, -1),
                 lambda: m.token_log_probs(w[:2], t, -100, 1), lambda: m.cross_entropy(w[:2], t, -100, True, 1.0)):
        with pytest.raises(RuntimeError):
            call()
    assert not m.clip_supported([w]) and not m.clip_supported([])
    assert m.clip_grads([w], False, 0, 1.0, 1.0, True) is None
    assert m.launch_counts() == {}
    with pytest.raises(TypeError):
        m.clip_grads([None], False, 0, 1.0, 1.0, True)


def test_counters_include_attached_sources():
    from mgwfbp_b200.ops import counters
    theirs = {'somewhere': 3}
    counters.attach(lambda: theirs)
    try:
        before = counters.snapshot()
        theirs['somewhere'] = 5
        counters.bump('here')
        assert counters.diff(before) == {'somewhere': 2, 'here': 1}
        kept = dict(counters._counts)
        counters.reset()
        assert counters.total() == 0 and counters.snapshot() == {}
        theirs['somewhere'] = 6
        assert counters.total() == 1
        counters._counts.clear()
        counters._counts.update(kept)
    finally:
        counters._sources.pop()
        counters._counts.pop('here', None)
