"""Plain numpy forms of the language-model operators on shares: exact words, 64-bit floats."""
import math

import numpy as np

U = np.uint64


def words(a):
    return np.asarray(a).astype(np.int64, copy=False).view(U)


def embed(T, vocab, dim, ids, scale, shift):
    T = words(T).reshape(vocab, dim)
    out = np.zeros((len(ids), dim), U)
    for t, i in enumerate(ids):
        if 0 <= i < vocab:
            out[t] = T[i] * U(scale % 2 ** 64)
    return (out.view(np.int64) >> shift).ravel()


def embed_grad(G, ids, vocab, dim, scale, shift):
    G = words(G).reshape(len(ids), dim)
    out = np.zeros((vocab, dim), U)
    for t, i in enumerate(ids):
        if 0 <= i < vocab:
            out[i] += G[t]
    return ((out * U(scale % 2 ** 64)).view(np.int64) >> shift).ravel()


def sqnorm(X0s, X1s, mask):
    z = sum((int(np.sum(words(a) * (words(a) + words(b) * U(2)), dtype=U)) for a, b in zip(X0s, X1s)), 0)
    z = (z + mask) % 2 ** 64
    return z - 2 ** 64 if z >= 2 ** 63 else z


def clip_factor(S, max_norm, number):
    if S == 0:
        return 2 ** number
    return min(2 ** number, math.isqrt((max_norm << number) ** 2 // S))


def opened(a, b, c):
    x = words(a).copy()
    for s in (b, c):
        if s is not None:
            x += words(s)
    return x.view(np.int64)


def logprobs(x, frac, ids, top):
    """x: rows x vocab opened words.  Returns logp, entropy, top_ids, top_logp, row_max, log_sum, and the 64-bit distances."""
    rows, vocab = x.shape
    m = x.max(1)
    d = (m[:, None].view(U) - x.view(U)).astype(np.float64) * 2.0 ** -frac
    e = np.exp(-d)
    S = e.sum(1)
    ls = np.log(S)
    H = ls + (d * e).sum(1) / S
    lp = -(d + ls[:, None])
    ok = (ids >= 0) & (ids < vocab)
    logp = np.where(ok, np.take_along_axis(lp, np.where(ok, ids, 0), 1), 0.0) if ids.shape[1] else np.zeros(ids.shape)
    order = np.argsort(~x, axis=1, kind="stable")[:, :top]  # ~x reverses the order of the words without overflow
    return logp, H, order, np.take_along_axis(lp, order, 1), m, ls


def logprobs_grad(x, frac, ids, d_logp, d_entropy, row_max, log_sum, entropy):
    """Also returns a bound of the rounding errors of a 32-bit evaluation of the same formula."""
    rows, vocab = x.shape
    d = (row_max[:, None].view(U) - x.view(U)).astype(np.float64) * 2.0 ** -frac
    lp = -(d + log_sum.astype(np.float64)[:, None])
    p = np.exp(lp)
    g = np.zeros((rows, vocab))
    mag = np.zeros((rows, vocab))
    ok = (ids >= 0) & (ids < vocab)
    w = np.where(ok, d_logp.astype(np.float64), 0.0)
    for t in range(ids.shape[1]):
        r = np.nonzero(ok[:, t])[0]
        np.add.at(g, (r, ids[r, t]), w[r, t])
        np.add.at(mag, (r, ids[r, t]), np.abs(w[r, t]))
    W, Wabs = w.sum(1)[:, None], np.abs(w).sum(1)[:, None]
    g = g - p * W
    # half a step each: the distance, the sum with log_sum, the exponential's argument scale (|lp| of them), exp itself
    # (two), the products; the sums over ids add one step per id
    k = ids.shape[1] + 1
    err = 2.0 ** -24 * (k * mag + p * (Wabs * (3 * np.abs(lp) + 8 + k)) + 2 * (mag + p * np.abs(W)))
    if d_entropy is not None:
        h, H = d_entropy.astype(np.float64)[:, None], entropy.astype(np.float64)[:, None]
        g = g - h * p * (lp + H)
        err = err + 2.0 ** -24 * np.abs(h) * p * ((3 * np.abs(lp) + 12) * np.abs(lp + H) + 4 * (np.abs(lp) + np.abs(H)))
    return g, err
