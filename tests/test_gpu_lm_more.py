"""More of the language-model operators (run with -m gpu on an MI355X): forms and arguments that test_gpu_lm.py does not reach.
Words exactly; floats within bounds derived there, half a step (2^-24) per 32-bit operation."""
import os
import re

import numpy as np
import pytest

import lm_reference as ref
import protocols as pr
from test_gpu_lm import KINDS, LOWEST, STEP, gpu, logprob_bounds, logit_rows, resident, rnd, share, tokens  # noqa: F401

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


# ---- forms that no other test reaches
def forward_form(rows, vocab):
    """Which form of the forward pass a call takes, by the rules and the limits of the kernels' source."""
    src = open(os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "mpc_amd", "csrc", "lm.hip")).read()
    limit = {k: int(v) for k, v in re.findall(r"\b(LP_\w+) = (\d+)[,;]", src)}
    splits = 1 if rows >= limit["LP_ROWS"] else limit["LP_GROUPS"] // rows
    splits = min(splits, -(-vocab // limit["LP_CHUNK"]))
    chunk = -(-(-(-vocab // splits)) // 2048) * 2048
    if -(-vocab // chunk) > 1:
        return "split"
    return "wave" if vocab <= 1024 or (vocab <= limit["LP_WAVE_ROW"] and rows >= 2048) else "workgroup"


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("form,rows,vocab,per_row,top,shares", [
    ("workgroup", 3, 1025, 1, 32, 3), ("workgroup", 2, 1500, 2, 5, 2), ("workgroup", 5, 2048, 1, 20, 3), ("workgroup", 1, 1537, 3, 0, 1),
    ("workgroup", 300, 2500, 1, 32, 3), ("workgroup", 257, 9001, 1, 5, 2), ("workgroup", 256, 4097, 300, 1, 1),
    ("wave", 2048, 1500, 1, 20, 3), ("wave", 2051, 1025, 2, 32, 2), ("wave", 2048, 8192, 1, 5, 1), ("split", 255, 4097, 1, 32, 2),
    ("split", 2, 2049, 1, 32, 3)])
def test_logprobs_of_every_form(gpu, kind, form, rows, vocab, per_row, top, shares):
    """One wavefront a row, one workgroup a row (a wavefront without words among them), several workgroups a row."""
    assert forward_form(rows, vocab) == form
    rng = np.random.default_rng(rows * 7 + vocab + KINDS.index(kind))
    x = logit_rows(kind, rng, rows, vocab, 16)
    ids = rng.integers(0, vocab, (rows, per_row))
    bad = rng.random(ids.shape) < 0.1
    ids[bad] = rng.choice(np.array([-1, vocab, LOWEST, 2 ** 40], np.int64), int(bad.sum()))
    got = gpu.reveal_logprobs(*share(rng, x, shares), rows, vocab, 16, ids.ravel(), top)
    want = ref.logprobs(x, 16, ids, top)
    logp, H, top_ids, top_logp, m, ls = [g.reshape(w.shape) for g, w in zip(got, want)]
    assert np.array_equal(m, want[4]) and np.array_equal(top_ids, want[2])
    d_ls, d_H = logprob_bounds(x, 16, want, vocab)
    assert (np.abs(ls - want[5]) <= d_ls).all() and (np.abs(H - want[1]) <= d_H).all()
    assert (np.abs(logp - want[0]) <= d_ls[:, None] + 3 * STEP * np.abs(want[0])).all()
    assert (np.abs(top_logp - want[3]) <= d_ls[:, None] + 3 * STEP * np.abs(want[3])).all()


def grad_bound(p, lp, w_abs, at_abs, h, H, k):
    """Half steps of the gradient's formula, as lm_reference.logprobs_grad counts them, on tensors."""
    return STEP * (k * at_abs + p * w_abs * (3 * lp.abs() + 8 + k) + 2 * (at_abs + p * w_abs)
                   + h.abs() * p * ((3 * lp.abs() + 12) * (lp + H).abs() + 4 * (lp.abs() + H.abs())))


@pytest.mark.parametrize("shares", [1, 2, 3])
def test_logprobs_grad_of_large_calls(resident, shares):
    """Calls beyond the last-level cache, whose stores do not stay in it: words of given ids are written a second time, by
    another wavefront.  Every word of the floats and of the ring words, an odd number of columns, ids at the ends of the
    workgroups' words, the same one several times, outside."""
    ctx, torch, dev, be, side = resident
    rows, vocab, k, frac, grad_frac = 1100, 32769, 6, 16, 30
    with torch.cuda.stream(side):
        x = (torch.randn(rows, vocab, device=dev) * 3 * 65536).long()
        parts = [torch.randint(-2 ** 63, 2 ** 63 - 1, (rows, vocab), device=dev) for _ in range(shares - 1)]
        first = x.clone()
        for s in parts:
            first -= s
        ids = torch.randint(0, vocab, (rows, k), device=dev)
        ids[:, 1] = torch.arange(rows, device=dev) % 17 * 2048  # a workgroup's first word, the last of the row among them
        ids[:, 2] = (torch.arange(rows, device=dev) % 16 + 1) * 2048 - 1  # its last
        ids[:, 4] = ids[:, 3]
        ids[::7, 5] = -1
        ids[1::7, 5] = ids[1::7, 0]
        w, h = torch.randn(rows, k, device=dev), torch.randn(rows, device=dev)
        m = x.amax(1)
        ls, H = torch.empty(rows, device=dev), torch.empty(rows, device=dev)
        for a in range(0, rows, 100):
            lp = torch.log_softmax(x[a:a + 100].double() / 2 ** frac, 1)
            ls[a:a + 100], H[a:a + 100] = -lp.amax(1).float(), -(lp.exp() * lp).sum(1).float()
        grad, words = torch.full((rows, vocab), np.nan, device=dev), torch.zeros(rows, vocab, dtype=torch.int64, device=dev)
        only = torch.full((rows, vocab), np.nan, device=dev)
        b, c = (parts + [None, None])[:2]
        ctx.call("reveal_logprobs_grad", first, b, c, rows, vocab, frac, ids, k, w, h, m, ls, H, grad, words, grad_frac)
        ctx.call("reveal_logprobs_grad", first, b, c, rows, vocab, frac, ids, k, w, h, m, ls, H, only, None, 0)
        assert torch.equal(only, grad)
        assert torch.equal(words, torch.round(grad.double() * 2.0 ** grad_frac).long())
        inside = ids >= 0
        live = torch.where(inside, w, 0).double()
        for a in range(0, rows, 100):
            s = slice(a, a + 100)
            lp = (x[s] - m[s, None]).double() / 2 ** frac - ls[s, None].double()
            p, W, Wabs = lp.exp(), live[s].sum(1, keepdim=True), live[s].abs().sum(1, keepdim=True)
            hh, HH = h[s, None].double(), H[s, None].double()
            at = torch.zeros_like(p).scatter_add_(1, ids[s].clamp(min=0), live[s])
            at_abs = torch.zeros_like(p).scatter_add_(1, ids[s].clamp(min=0), live[s].abs())
            want = at - p * W - hh * p * (lp + HH)
            assert ((grad[s] - want).abs() <= grad_bound(p, lp, Wabs, at_abs, hh, HH, k + 1) + 1e-37).all(), a
        del x, parts, first, grad, words, only
        torch.cuda.empty_cache()


def test_logprobs_grad_of_split_rows_beyond_one_launch(resident):
    """Rows of two workgroups each, more of them than one launch takes: the rows around the second launch's first one exactly,
    and every row's gradient adds up to nothing."""
    ctx, torch, dev, be, side = resident
    rows, vocab, frac = (1 << 21) + 3, 2049, 16
    with torch.cuda.stream(side):
        row = (torch.randn(vocab, device=dev) * 3 * 65536).long()
        x = row.repeat(rows, 1)
        x += torch.arange(rows, device=dev)[:, None]  # the same distribution, another largest word
        ids = (torch.arange(rows, device=dev) * 7 % vocab)[:, None].contiguous()
        w = torch.rand(rows, 1, device=dev) + 0.5
        m, ls = row.amax() + torch.arange(rows, device=dev), torch.logsumexp((row - row.amax()).double() / 2 ** frac, 0).float().repeat(rows)
        lp = (row - row.amax()).double() / 2 ** frac - ls[0].double()
        grad = torch.empty(rows, vocab, device=dev)
        ctx.call("reveal_logprobs_grad", x, None, None, rows, vocab, frac, ids, 1, w, None, m, ls, None, grad, None, 0)
        zero = torch.zeros((), dtype=torch.float64, device=dev)
        for a, b in ((0, 64), ((1 << 21) - 64, rows)):
            at = torch.zeros(b - a, vocab, dtype=torch.float64, device=dev).scatter_add_(1, ids[a:b], w[a:b].double())
            p = lp.exp()[None]
            assert ((grad[a:b] - (at - p * w[a:b].double())).abs() <= grad_bound(p, lp[None], w[a:b].double(), at, zero, zero, 2) + 1e-37).all()
        # the rounding errors of a row's words together (weights up to 1.5), and that of log_sum, of |log_sum| steps in all p
        most = 1.5 * STEP * ((lp.exp() * (3 * lp.abs() + 12)).sum() + 4 + ls[0].abs()).item()
        for a in range(0, rows, 1 << 18):
            assert (grad[a:a + (1 << 18)].double().sum(1).abs() <= most).all()
        del x, grad
        torch.cuda.empty_cache()


@pytest.mark.parametrize("shares", [1, 2])
@pytest.mark.parametrize("vocab,dim,n,kind", [(9000, 33, 5000, "zipf"), (40000, 130, 3000, "one"), (70000, 5, 40000, "zipf"),
                                              (70000, 130, 33000, "one"), (9000, 8, 2100, "none")])
def test_embed_grad_accumulates_few_tokens_of_many_rows(gpu, shares, vocab, dim, n, kind):
    """Fewer tokens than rows, more than the one-launch form takes, frequent ones among them: added to what is there, and rows
    without tokens stay as they were."""
    ctx = gpu.ctx
    rng = np.random.default_rng(vocab + dim + n)
    ids = tokens(rng, n, vocab, kind)
    if kind == "zipf":
        assert np.bincount(ids[(ids >= 0) & (ids < vocab)]).max() > 32
    G, old = [rnd(rng, n, dim) for _ in range(shares)], [rnd(rng, vocab * dim + 16) for _ in range(shares)]
    dG, dT, dI = [ctx.to_device(g.ravel()) for g in G], [ctx.to_device(o) for o in old], ctx.to_device(ids)
    scale, shift = (77777, 16) if shares == 1 else (-12345, 0)
    ws = ctx.empty(np.uint8, ctx.scratch_bytes("ring_embed_grad", n, vocab, dim))
    ctx.call("ring_embed_grad", dG[0], dG[1] if shares == 2 else None, dI, n, vocab, dim, scale, shift, 1, ws, dT[0],
             dT[1] if shares == 2 else None)
    ctx.sync()
    ok = (ids >= 0) & (ids < vocab)
    for k in range(shares):
        add = np.zeros((vocab, dim), np.uint64)
        np.add.at(add, ids[ok], ref.words(G[k])[ok])
        add = ((add * np.uint64(scale % 2 ** 64)).view(np.int64) >> shift).ravel()
        want = old[k].copy()
        want[:vocab * dim] = (ref.words(want[:vocab * dim]) + ref.words(add)).view(np.int64)
        assert np.array_equal(dT[k].to_host(), want), k


def test_clipping_of_norms_beyond_the_opened_word(gpu, orc):
    """A norm of 2^32 words and more wraps in the opened word; truncated by k bits first, the tensors are clipped as they should
    be (the way that mpcx_aby3_clip_local and ABY3Engine::clip_norm name)."""
    frac, k = 16, 8
    rng = np.random.default_rng(3)
    X = [rng.normal(size=n) * 9000 for n in (100, 7, 400)]  # reals of norm 2e5
    X = [(x * 2 ** frac).astype(np.int64) for x in X]
    assert sum(int(v) ** 2 for x in X for v in x) >= 2 ** 64
    w = pr.World(gpu)
    shares = [pr.aby3_trunc(w, pr.aby3_share(w, x, x.size), k) for x in X]
    open3 = lambda S: (ref.words(S[0][0]) + ref.words(S[1][0]) + ref.words(S[2][0])).view(np.int64)
    cut = np.concatenate([open3(s) for s in shares])
    S = sum(int(v) ** 2 for v in cut)
    assert S < 2 ** 64 and np.abs(cut - (np.concatenate(X) >> k)).max() <= 1
    clipped, coef = pr.aby3_clip(w, shares, (20000 << frac) >> k, frac - k)  # to a norm of 20000
    c = ref.clip_factor(S, 20000 << (frac - k), frac - k)
    assert int(coef[0]) == c and 0 < c < 2 ** (frac - k)
    got = open3(clipped)
    assert np.abs(got - ((cut * c) >> (frac - k))).max() <= 2
    assert np.sqrt((got.astype(np.float64) ** 2).sum()) <= (20000 << (frac - k)) + 2 * np.sqrt(got.size)
