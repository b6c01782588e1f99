"""More of the language-model operators (run with -m gpu on an MI355X): forms and arguments that test_gpu_lm.py does not reach.
Words exactly; floats within bounds derived there, half a step (2^-24) per 32-bit operation."""
import numpy as np
import pytest

import lm_reference as ref
from test_gpu_lm import LOWEST, STEP, gpu, logit_rows, resident, rnd, share, tokens  # noqa: F401

pytestmark = pytest.mark.gpu


def test_logprobs_grad_of_masked_words_under_large_weights(gpu):
    """A masked word has probability 0, and its gradient is what is given for it and nothing else, however far away it lies and
    however large the weights are (the product of the weight and ln p is beyond the floats)."""
    rows, vocab, frac = 3, 70, 0
    x = np.full((rows, vocab), LOWEST, np.int64)
    x[:, 5], x[:, 6] = 100, 99
    ids = np.array([[9], [5], [-1]])
    _, H, _, _, m, ls = ref.logprobs(x, frac, ids, 0)
    w, h = np.full((rows, 1), 2.0, np.float32), np.full(rows, 1e25, np.float32)
    grad, _ = gpu.reveal_logprobs_grad(x.ravel(), None, None, rows, vocab, frac, ids.ravel(), w.ravel(), h, m, ls.astype(np.float32),
                                       H.astype(np.float32), 20)
    grad = grad.reshape(rows, vocab)
    masked = np.ones(vocab, bool)
    masked[5:7] = False
    want = np.zeros((rows, vocab), np.float32)
    want[0, 9] = 2
    assert np.array_equal(grad[:, masked], want[:, masked])
    assert np.isfinite(grad).all() and (np.abs(grad[:, 5:7]) > 1e23).all()


@pytest.mark.parametrize("rows,vocab,per_row,shares,kind", [
    (3, 5, 32, 1, "few"), (3, 5, 33, 2, "few"), (5, 700, 33, 3, "any"), (2, 768, 1000, 1, "any"), (9, 64, 64, 2, "every"),
    (2, 769, 65, 3, "any"), (3, 2047, 100, 1, "edges"), (2, 2048, 129, 2, "edges"), (2, 6145, 4097, 3, "edges"), (4, 3000, 300, 3, "one"),
    (2, 700, 129, 1, "one"), (3, 40, 90, 3, "none"), (2, 5000, 5000, 2, "every")])
def test_logprobs_grad_of_many_ids(gpu, rows, vocab, per_row, shares, kind):
    """Rows of more ids than a few: all different, many times the same one, at the ends of a workgroup's words, outside."""
    rng = np.random.default_rng(rows + vocab + per_row)
    frac, grad_frac, f32 = 16, 20, np.float32
    x = logit_rows("normal", rng, rows, vocab, frac)
    ids = rng.integers(0, vocab, (rows, per_row))
    if kind == "few":
        ids = rng.integers(0, 2, (rows, per_row))
    elif kind == "every":
        ids = np.stack([rng.permutation(vocab) for _ in range(rows)])
    elif kind == "one":
        ids[:] = vocab - 1
    elif kind == "edges":
        at = np.array([e for e in (0, 1, 767, 768, 2046, 2047, 2048, 4095, 4096, 6143, 6144, vocab - 1) if e < vocab])
        ids[:, ::3] = rng.choice(at, ids[:, ::3].shape)
    bad = rng.random(ids.shape) < (1.0 if kind == "none" else 0.1)
    ids[bad] = rng.choice(np.array([-1, vocab, LOWEST, 2 ** 40, 2 ** 32], np.int64), int(bad.sum()))
    _, H, _, _, m, ls = ref.logprobs(x, frac, ids, 0)
    H, ls = H.astype(f32), ls.astype(f32)
    d_logp, d_ent = rng.normal(size=ids.shape).astype(f32), rng.normal(size=rows).astype(f32)
    d_logp[bad] = np.nan  # what is given for an id outside is not looked at
    grad, words = gpu.reveal_logprobs_grad(*share(rng, x, shares), rows, vocab, frac, ids.ravel(), d_logp.ravel(), d_ent, m, ls, H, grad_frac)
    want, err = ref.logprobs_grad(x, frac, ids, np.where(bad, 0, d_logp).astype(f32), d_ent, m, ls, H)
    grad = grad.reshape(rows, vocab)
    assert (np.abs(grad - want) <= err + 1e-37).all(), np.abs(grad - want).max()
    assert np.array_equal(words.reshape(rows, vocab), np.rint(grad.astype(np.float64) * 2.0 ** grad_frac).astype(np.int64))


def test_logprobs_grad_of_a_dense_target_distribution(resident):
    """As many ids as words: the work grows with their number, not with its square (0.3 ms; the square would take 400)."""
    ctx, torch, dev, be, side = resident
    rows, vocab = 16, 32768
    with torch.cuda.stream(side):
        x = (torch.randn(rows, vocab, device=dev) * 3 * 65536).long()
        ids = torch.arange(vocab, device=dev).flip(0).repeat(rows, 1)
        w = torch.softmax(torch.randn(rows, vocab, device=dev), 1)
        m = x.amax(1)
        lp = torch.log_softmax(x.double() / 65536, 1)
        ls = (-lp.amax(1)).float()
        grad = torch.empty(rows, vocab, device=dev)
        call = lambda: ctx.call("reveal_logprobs_grad", x, None, None, rows, vocab, 16, ids, vocab, w, None, m, ls, None, grad, None, 0)
        call()
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        call()
        end.record()
        side.synchronize()
        assert start.elapsed_time(end) < 20
        p, W = torch.exp(lp), w.double().sum(1, keepdim=True)
        want = w.double().flip(1) - p * W
        # the sum of the weights (32768 / 256 of them one after the other, then a tree) and the terms of one word
        bound = STEP * (w.double().flip(1) + p * W * (vocab / 256 + 10 + 3 * lp.abs() + 12) + 2 * want.abs())
        assert ((grad - want).abs() <= bound + 1e-37).all()
