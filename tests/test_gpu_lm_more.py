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
