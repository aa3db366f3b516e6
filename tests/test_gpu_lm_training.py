"""The language-model operators where the framework calls them: the PTB model's embedding and loss, clipping under
optimizers that the fused update does not cover, and the report of a word outside the vocabulary."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _trainer(**kw):
    from mgwfbp_b200.trainer import DLTrainer
    args = dict(dist=False, batch_size=4, data_dir='synthetic', dataset='ptb', dnn='lstm', lr=1.0, nworkers=1, num_steps=6, seed=3)
    args.update(kw)
    return DLTrainer(0, 1, **args)


def test_ptb_model_with_and_without_the_operators(monkeypatch):
    """Same seed, same batch: loss and gradients with the operators are those of torch's embedding and criterion."""
    from mgwfbp_b200 import settings
    from mgwfbp_b200.ops import counters
    from mgwfbp_b200.ops.embedding import FusedEmbedding
    from mgwfbp_b200.ops.logprob import FusedCrossEntropyLoss
    prev = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    try:
        results = []
        for on in (True, False):
            monkeypatch.setattr(settings, 'FUSE_LM_OPS', on)
            t = _trainer()
            assert isinstance(t.net.word_embeddings, FusedEmbedding) == on
            assert isinstance(t.criterion, FusedCrossEntropyLoss) == on
            t.net.eval()                                  # no dropout: both runs compute the same function
            batch = t.to_device(t.data_iter())
            before = counters.snapshot()
            loss, outputs, labels, _ = t.forward_loss(batch, None, on_device=True)
            t.backward(loss)
            seen = counters.diff(before)
            assert (seen.get('embedding_grad', 0) == 1 and seen.get('cross_entropy_fwd', 0) == 1) == on
            results.append((loss.detach(), {n: p.grad.clone() for n, p in t.net.named_parameters()}))
    finally:
        torch.backends.cuda.matmul.allow_tf32 = prev
    (la, ga), (lb, gb) = results
    torch.testing.assert_close(la, lb, rtol=1e-5, atol=1e-6)
    assert list(ga) == list(gb)
    for n in ga:
        scale = float(gb[n].abs().max())
        assert float((ga[n] - gb[n]).abs().max()) <= 1e-4 * scale, n


def test_ptb_evaluation_reports_next_word_statistics():
    t = _trainer()
    perplexity = t.test(0)
    assert perplexity > 1.0
    w = t.word_stats
    # an untrained model: nearly uniform over 10000 words (entropy at most ln 10000 = 9.2103)
    assert 0.0 <= w['top1'] <= w['top5'] <= 100.0 and 8.0 < w['entropy'] <= 9.2104


def test_word_outside_the_vocabulary_stops_the_step():
    import mgwfbp_b200 as hvd
    from mgwfbp_b200.engine import TrainStep
    from mgwfbp_b200.ops._tokens import TokenIndexError, check_status
    t = _trainer()
    t.update_optimizer(hvd.DistributedOptimizer(t.optimizer, named_parameters=t.net.named_parameters(), norm_clip=0.25))
    step = TrainStep(t, use_graph=False)
    inputs, labels = t.data_iter()
    check_status()
    inputs = inputs.clone()
    inputs[1, 2] = t.net.vocab_size
    with pytest.raises(TokenIndexError, match='outside the vocabulary'):
        step.run((inputs, labels))
        torch.cuda.synchronize()
        step.drain()
    check_status()


def test_ptb_steps_replayed_from_a_graph():
    """Eager and replayed steps run the operators; the clip keeps every update within lr * 0.25."""
    import mgwfbp_b200 as hvd
    from mgwfbp_b200.engine import TrainStep
    from mgwfbp_b200.ops import counters
    t = _trainer(lr=2.0)
    t.update_optimizer(hvd.DistributedOptimizer(t.optimizer, named_parameters=t.net.named_parameters(), norm_clip=0.25))
    step = TrainStep(t)
    before = counters.snapshot()
    for i in range(7):
        w = t.net.word_embeddings.weight.detach().clone()
        step.run(t.data_iter())
        torch.cuda.synchronize()
        moved = float((t.net.word_embeddings.weight.detach() - w).double().norm())
        assert 0.0 < moved <= 2.0 * 0.25 * 1.001
    step.drain()
    assert all(l == l for l in step.losses) and step.graphed
    seen = counters.diff(before)
    # seven steps, and the capture, whose calls are counted although they only record
    assert seen['embedding_grad'] == seen['cross_entropy_fwd'] == 8


@pytest.mark.parametrize('make', [lambda ps: torch.optim.Adam(ps, lr=0.01), lambda ps: torch.optim.RMSprop(ps, lr=0.01)],
                         ids=['adam', 'rmsprop'])
def test_clipping_under_other_optimizers(make):
    import mgwfbp_b200 as hvd
    from mgwfbp_b200.ops import counters
    torch.manual_seed(0)
    sizes = [(30, 7), (5,), (64, 33)]
    mine = [torch.nn.Parameter(torch.randn(s, device='cuda')) for s in sizes]
    theirs = [torch.nn.Parameter(p.detach().clone()) for p in mine]
    opt = hvd.DistributedOptimizer(make(mine), named_parameters=[('p%d' % i, p) for i, p in enumerate(mine)], norm_clip=0.25)
    opt.set_grad_scale(0.5)
    ref = make(theirs)
    for _ in range(3):
        for p, q in zip(mine, theirs):
            p.grad = torch.randn_like(p)
            q.grad = p.grad * 0.5
        before = counters.snapshot()
        opt.step()
        assert counters.diff(before).get('grad_scale') == 1
        torch.nn.utils.clip_grad_norm_(theirs, 0.25)
        ref.step()
    for p, q in zip(mine, theirs):
        torch.testing.assert_close(p, q, rtol=1e-5, atol=1e-6)
