"""Language-model operators on secret shares (run with -m gpu on an MI355X) against plain numpy forms: words exactly,
floats within bounds derived from half a step (2^-24) per 32-bit operation."""
import ctypes

import numpy as np
import pytest

import lm_reference as ref
import protocols as pr
from oracle_lib import KEY01, KEY12, KEY20, prg_pops

pytestmark = pytest.mark.gpu
STEP = 2.0 ** -24
LOWEST, HIGHEST = -2 ** 63, 2 ** 63 - 1


@pytest.fixture(scope="module")
def gpu():
    from backends import GpuBackend
    return GpuBackend()


@pytest.fixture(scope="module")
def resident():
    """A context on a torch stream, arrays as torch tensors."""
    import torch
    from backends import ResidentBackend
    from mpc_amd import Context
    dev = torch.device("cuda", 0)
    ctx = Context(0)
    side = torch.cuda.Stream(dev)
    ctx.call("set_stream", side.cuda_stream)
    yield ctx, torch, dev, ResidentBackend(ctx, torch, dev), side
    torch.cuda.synchronize()
    ctx.close()
    torch.cuda.empty_cache()


def rnd(rng, *shape):
    return rng.integers(LOWEST, 2 ** 63, shape, dtype=np.int64)


def tokens(rng, n, vocab, kind="zipf"):
    if kind == "one":  # every token the same
        ids = np.full(n, vocab // 2, np.int64)
    elif kind == "none":  # nothing but padding
        ids = np.full(n, -1, np.int64)
    else:
        ids = np.minimum((vocab ** rng.random(n)).astype(np.int64), vocab) - 1
        ids = ids * 7919 % vocab
        bad = rng.random(n) < 0.05
        ids[bad] = rng.choice(np.array([-1, vocab, LOWEST, HIGHEST, 2 ** 32, 2 ** 40], np.int64), int(bad.sum()))
    return ids


# ------------------------------------------------------------------ lookup and its gradient
@pytest.mark.parametrize("vocab,dim,n", [(1, 1, 1), (5, 1, 7), (7, 3, 100), (1009, 129, 257), (64, 256, 1000), (300, 515, 33),
                                         (10, 1024, 5), (3, 2048, 3), (40, 64, 0), (2000, 31, 1)])
@pytest.mark.parametrize("shares", [1, 2])
def test_embed(gpu, vocab, dim, n, shares):
    rng = np.random.default_rng(vocab * 31 + dim * 7 + n)
    ids = tokens(rng, n, vocab)
    T = [rnd(rng, vocab * dim) for _ in range(shares)]
    for scale, shift in ((1, 0), (-3, 0), (0x123456789ABCDEF, 0)) + (((1487181, 16), (5, 63)) if shares == 1 else ()):
        got = gpu.ring_embed(T[0], T[1] if shares == 2 else None, vocab, dim, ids, scale, shift)
        for k, g in enumerate([got] if shares == 1 else got):
            assert np.array_equal(g, ref.embed(T[k], vocab, dim, ids, scale, shift)), (scale, shift, k)


@pytest.mark.parametrize("vocab,dim,n", [(1, 1, 1), (5, 1, 700), (7, 3, 100), (1009, 129, 257), (64, 256, 3000), (300, 515, 33),
                                         (10, 1024, 5), (4, 700, 9000), (40, 64, 0), (2000, 31, 1), (70001, 2, 500)])
@pytest.mark.parametrize("kind", ["zipf", "one", "none"])
@pytest.mark.parametrize("shares", [1, 2])
def test_embed_grad(gpu, vocab, dim, n, kind, shares):
    rng = np.random.default_rng(vocab * 31 + dim * 7 + n)
    ids = tokens(rng, n, vocab, kind)
    G = [rnd(rng, n * dim) for _ in range(shares)]
    for scale, shift in ((1, 0), (0x123456789ABCDEF, 0)) + (((1487181, 16),) if shares == 1 else ()):
        got = gpu.ring_embed_grad(G[0], G[1] if shares == 2 else None, ids, vocab, dim, scale, shift)
        for k, g in enumerate([got] if shares == 1 else got):
            assert np.array_equal(g, ref.embed_grad(G[k], ids, vocab, dim, scale, shift)), (scale, shift, k)


@pytest.mark.parametrize("vocab,dim,n,kind", [(300, 130, 5000, "zipf"), (300, 130, 5000, "one"), (9000, 40, 140001, "zipf"),
                                              (3, 200, 140001, "zipf"), (1100000, 2, 70, "zipf"), (1100000, 2, 5000, "one"),
                                              (33, 1030, 4100, "cycle"), (33, 257, 33 * 32, "cycle"), (33, 257, 33 * 33, "cycle"),
                                              (700, 129, 40000, "cycle"), (20, 5, 6000, "none"), (5000, 300, 4097, "zipf")])
@pytest.mark.parametrize("shares", [1, 2])
def test_embed_grad_of_many_tokens(gpu, vocab, dim, n, kind, shares):
    """Rows of 32, 33, .. tokens at every place of the order, texts of one token, vocabularies and lengths of every form."""
    rng = np.random.default_rng(n + vocab)
    ids = np.arange(n, dtype=np.int64) % vocab if kind == "cycle" else tokens(rng, n, vocab, kind)
    G = [rnd(rng, n, dim) for _ in range(shares)]
    got = gpu.ring_embed_grad(G[0].ravel(), G[1].ravel() if shares == 2 else None, ids, vocab, dim, -7, 0)
    ok = (ids >= 0) & (ids < vocab)
    for k, g in enumerate([got] if shares == 1 else got):
        want = np.zeros((vocab, dim), np.uint64)
        np.add.at(want, ids[ok], ref.words(G[k])[ok])
        assert np.array_equal(ref.words(g).reshape(vocab, dim), want * np.uint64(2 ** 64 - 7)), k


@pytest.mark.parametrize("shares", [1, 2])
@pytest.mark.parametrize("vocab,dim,n", [(300, 130, 2000), (5, 1, 4000), (9000, 33, 40), (20, 8, 0)])
def test_embed_grad_accumulates(gpu, shares, vocab, dim, n):
    """accumulate adds to what is there, and leaves the rows that no token names as they were; the words behind the last
    row stay what they were too."""
    ctx = gpu.ctx
    rng = np.random.default_rng(vocab + dim)
    ids = tokens(rng, n, vocab)
    G = [rnd(rng, n * dim) for _ in range(shares)]
    old = [rnd(rng, vocab * dim + 16) for _ in range(shares)]
    dG, dT, dI = [ctx.to_device(g) for g in G], [ctx.to_device(o) for o in old], ctx.to_device(ids)
    scale, shift = (77777, 16) if shares == 1 else (-12345, 0)
    ws = ctx.empty(np.uint8, ctx.scratch_bytes("ring_embed_grad", n, vocab, dim))
    ctx.call("ring_embed_grad", dG[0], dG[1] if shares == 2 else None, dI, n, vocab, dim, scale, shift, 1, ws, dT[0],
             dT[1] if shares == 2 else None)
    ctx.sync()
    for k in range(shares):
        got = dT[k].to_host()
        want = old[k].copy()
        want[:vocab * dim] = (ref.words(want[:vocab * dim]) + ref.words(ref.embed_grad(G[k], ids, vocab, dim, scale, shift))).view(np.int64)
        assert np.array_equal(got, want), k


def test_embed_and_gradient_at_unaligned_addresses(gpu):
    """Arrays that start 8 bytes behind a 16-byte boundary, outputs as well."""
    ctx = gpu.ctx
    rng = np.random.default_rng(8)
    for vocab, dim, n in ((33, 64, 50), (33, 65, 50), (7, 512, 300)):
        ids = tokens(rng, n, vocab)
        T, G = rnd(rng, vocab * dim), rnd(rng, n * dim)
        at = lambda a: ctx.to_device(np.concatenate([np.zeros(1, np.int64), a])).view(1, a.size)
        E, D = ctx.empty(np.int64, n * dim + 1), ctx.empty(np.int64, vocab * dim + 1)
        E1, D1 = E.view(1, n * dim), D.view(1, vocab * dim)
        ws = ctx.empty(np.uint8, ctx.scratch_bytes("ring_embed_grad", n, vocab, dim))
        ctx.call("ring_embed", at(T), None, vocab, dim, at(ids), n, 3, 0, E1, None)
        ctx.call("ring_embed_grad", at(G), None, at(ids), n, vocab, dim, 3, 0, 0, ws, D1, None)
        ctx.sync()
        assert np.array_equal(E1.to_host(), ref.embed(T, vocab, dim, ids, 3, 0))
        assert np.array_equal(D1.to_host(), ref.embed_grad(G, ids, vocab, dim, 3, 0))


def test_scratch_memory_may_begin_at_any_word(gpu):
    """Scratch memory 8 bytes behind a 16-byte boundary, and the words behind its end are left as they were."""
    ctx = gpu.ctx
    rng = np.random.default_rng(31)

    def scratch(name, *sizes):
        size = ctx.scratch_bytes(name, *sizes)
        assert size % 8 == 0
        whole = ctx.to_device(np.full(size // 8 + 9, 0x5A5A, np.int64))
        return whole, whole.view(1, size // 8), size // 8

    def untouched(whole, words):
        h = whole.to_host()
        return h[0] == 0x5A5A and (h[1 + words:] == 0x5A5A).all()

    for vocab, dim, n in ((9000, 33, 3000), (70, 130, 5000), (40000, 64, 40000)):
        ids, G = tokens(rng, n, vocab), [rnd(rng, n * dim) for _ in range(2)]
        whole, ws, words = scratch("ring_embed_grad", n, vocab, dim)
        D = [ctx.empty(np.int64, vocab * dim) for _ in range(2)]
        dG, dI = [ctx.to_device(g) for g in G], ctx.to_device(ids)
        ctx.call("ring_embed_grad", dG[0], dG[1], dI, n, vocab, dim, 3, 0, 0, ws, D[0], D[1])
        ctx.sync()
        for k in range(2):
            assert np.array_equal(D[k].to_host(), ref.embed_grad(G[k], ids, vocab, dim, 3, 0))
        assert untouched(whole, words)
    for rows, vocab, top in ((1, 50000, 7), (5, 9001, 0), (300, 700, 3)):
        x = (rng.normal(size=(rows, vocab)) * 65536).astype(np.int64)
        whole, ws, words = scratch("reveal_logprobs", rows, vocab, top)
        dX, m, ti, tl = ctx.to_device(x), ctx.empty(np.int64, rows), ctx.empty(np.int64, rows * max(top, 1)), ctx.empty(np.float32, rows * max(top, 1))
        ctx.call("reveal_logprobs", dX, None, None, rows, vocab, 16, None, 0, top, ws, None, None, ti if top else None,
                 tl if top else None, m, None)
        ctx.sync()
        assert np.array_equal(m.to_host(), x.max(1))
        if top:
            assert np.array_equal(ti.to_host().reshape(rows, top), np.argsort(-x, axis=1, kind="stable")[:, :top])
        assert untouched(whole, words)
    X = [rnd(rng, 5000 + k) for k in range(200)]
    dX = [ctx.to_device(x) for x in X]
    whole, ws, words = scratch("aby3_sqnorm", 200)
    z = ctx.empty(np.int64, 1)
    ctx.call("aby3_sqnorm_local", dX, dX, [x.size for x in X], 200, KEY12, 3, KEY12, 3, ws, z)
    ctx.sync()
    with np.errstate(over="ignore"):
        assert int(z.to_host()[0]) == int(sum((3 * x * x).sum() for x in X))  # the two masks are the same word
    assert untouched(whole, words)


def test_embed_gradient_is_the_lookups_adjoint(gpu):
    """sum(G * embed(T)) = sum(embed_grad(G) * T) mod 2^64, and the difference quotient of the lookup in a direction is its
    value there (the map is linear, so the quotient is exact)."""
    rng = np.random.default_rng(2)
    vocab, dim, n = 211, 77, 640
    ids = tokens(rng, n, vocab)
    T, D, G = rnd(rng, vocab * dim), rnd(rng, vocab * dim), rnd(rng, n * dim)
    E = lambda t: ref.words(gpu.ring_embed(t, None, vocab, dim, ids, 9))
    dT = ref.words(gpu.ring_embed_grad(G, None, ids, vocab, dim, 9))
    lhs = np.sum(ref.words(G) * (E((ref.words(T) + ref.words(D)).view(np.int64)) - E(T)), dtype=np.uint64)
    assert lhs == np.sum(dT * ref.words(D), dtype=np.uint64)


def test_embed_reaches_rows_beyond_four_billion_words(resident):
    ctx, torch, dev, be, side = resident
    vocab, dim = (1 << 22) + 5, 1024
    with torch.cuda.stream(side):
        T = torch.empty(vocab * dim, dtype=torch.int64, device=dev)
        ids = torch.tensor([vocab - 1, 0, vocab - 3, vocab], dtype=torch.int64, device=dev)
        for i in ids[:3].tolist():
            T[i * dim:(i + 1) * dim] = torch.arange(dim, device=dev) + i
        E = torch.empty(4 * dim, dtype=torch.int64, device=dev)
        ctx.call("ring_embed", T, None, vocab, dim, ids, 4, 2, 0, E, None)
        want = torch.cat([(torch.arange(dim, device=dev) + i) * 2 for i in ids[:3].tolist()] + [torch.zeros(dim, dtype=torch.int64, device=dev)])
        assert torch.equal(E, want)
        # the gradient of the same table, in its place
        ws = torch.empty(ctx.scratch_bytes("ring_embed_grad", 4, vocab, dim), dtype=torch.uint8, device=dev)
        ctx.call("ring_embed_grad", E, None, ids, 4, vocab, dim, 1, 0, 0, ws, T, None)
        side.synchronize()
        for i in (vocab - 1, 0, vocab - 3):
            assert torch.equal(T[i * dim:(i + 1) * dim], (torch.arange(dim, device=dev) + i) * 2)
        for i in (1, 1 << 21, vocab - 2, vocab - 4):
            assert not T[i * dim:(i + 1) * dim].any()
        del T, ws
        torch.cuda.empty_cache()


@pytest.mark.parametrize("dim,offset", [(1001, 0), (951, 3), (1024, 0), (1024, 1), (1024, 8), (250, 5)])
@pytest.mark.parametrize("shares", [1, 2])
def test_large_calls_at_any_line_offset(resident, dim, offset, shares):
    """Calls beyond the last-level cache, whose stores go by whole lines: rows that begin anywhere in one, and the words
    before the first row and behind the last stay as they were."""
    ctx, torch, dev, _, side = resident
    with torch.cuda.stream(side):
        vocab, n = (300 << 20) // (8 * dim * shares), 37
        big = vocab + 1111
        words = lambda k: torch.randint(-2 ** 63, 2 ** 63 - 1, (k,), dtype=torch.int64, device=dev)
        put = lambda x: torch.cat([torch.zeros(offset, dtype=torch.int64, device=dev), x])[offset:]
        ids = torch.randint(0, vocab, (n,), dtype=torch.int64, device=dev)
        ids[5], ids[6:20] = vocab, ids[20]
        G = [words(n * dim) for _ in range(shares)]
        D = [words(vocab * dim + offset + 40) for _ in range(shares)]
        for accumulate in (0, 1):
            old = [d.clone() for d in D]
            ws = torch.empty(ctx.scratch_bytes("ring_embed_grad", n, vocab, dim), dtype=torch.uint8, device=dev)
            ctx.call("ring_embed_grad", G[0], G[1] if shares == 2 else None, ids, n, vocab, dim, 5, 0, accumulate, ws, D[0][offset:],
                     D[1][offset:] if shares == 2 else None)
            ok = ids < vocab
            for k in range(shares):
                want = old[k].clone()
                rows = want[offset:offset + vocab * dim].view(vocab, dim)
                if not accumulate:
                    rows.zero_()
                rows.index_add_(0, ids[ok], G[k].view(n, dim)[ok] * 5)
                assert torch.equal(D[k], want), (accumulate, k)
        # every row of the table, and some again
        some = torch.cat([torch.randperm(vocab, device=dev), torch.randint(0, vocab, (1111,), device=dev)])
        some[77] = -1
        E = [words(big * dim + offset + 40) for _ in range(shares)]
        old = [e.clone() for e in E]
        T = [put(d[:vocab * dim]) for d in D]
        ctx.call("ring_embed", T[0], T[1] if shares == 2 else None, vocab, dim, some, big, 3, 0, E[0][offset:],
                 E[1][offset:] if shares == 2 else None)
        for k in range(shares):
            rows = old[k][offset:offset + big * dim].view(big, dim)
            rows.copy_(T[k].view(vocab, dim)[some.clamp(min=0)] * 3)
            rows[77].zero_()
            assert torch.equal(E[k], old[k]), k
        del D, E, T, old, rows, want
        torch.cuda.empty_cache()


# ------------------------------------------------------------------ norm and clipping
LENS = [[1], [5], [0], [0, 3, 0], [4096], [4097, 1, 70000], [1] * 7, list(range(1, 301)), [257] * 130 + [0] * 3 + [300001],
        [784 * 128, 128, 128 * 128, 128, 128 * 10, 10]]


@pytest.mark.parametrize("lens", LENS, ids=lambda v: f"{len(v)}x{max(v)}")
def test_sqnorm(gpu, lens):
    rng = np.random.default_rng(sum(lens) + len(lens))
    X0, X1 = [rnd(rng, n) for n in lens], [rnd(rng, n) for n in lens]
    for pop_n, pop_p in ((0, 0), (63, 64), (1000, 7)):
        z = gpu.aby3_sqnorm_local(X0, X1, KEY01, pop_n, KEY20, pop_p)
        mask = int(prg_pops(KEY01, pop_n, 1)[0]) - int(prg_pops(KEY20, pop_p, 1)[0])
        assert int(z[0]) == ref.sqnorm(X0, X1, mask)


def test_sqnorm_of_no_tensors_is_the_mask(gpu):
    z = gpu.aby3_sqnorm_local([], [], KEY01, 3, KEY20, 4)
    assert int(z[0]) == ref.sqnorm([], [], int(prg_pops(KEY01, 3, 1)[0]) - int(prg_pops(KEY20, 4, 1)[0]))


def test_sqnorm_at_unaligned_addresses(gpu):
    ctx = gpu.ctx
    rng = np.random.default_rng(3)
    X0, X1 = [rnd(rng, n) for n in (1001, 64, 4096)], [rnd(rng, n) for n in (1001, 64, 4096)]
    at = lambda a, k: ctx.to_device(np.concatenate([np.zeros(k, np.int64), a])).view(k, a.size)
    z = ctx.empty(np.int64, 1)
    ws = ctx.empty(np.uint8, ctx.scratch_bytes("aby3_sqnorm", 3))
    a0, a1 = [at(x, 1) for x in X0], [at(x, k) for k, x in enumerate(X1)]
    ctx.call("aby3_sqnorm_local", a0, a1, [x.size for x in X0], 3, KEY01, 0, KEY01, 0, ws, z)
    ctx.sync()
    assert int(z.to_host()[0]) == ref.sqnorm(X0, X1, 0)


def test_sqnorm_of_a_tensor_beyond_four_billion_words(resident):
    ctx, torch, dev, be, side = resident
    n = (1 << 32) + 77
    with torch.cuda.stream(side):
        x0 = torch.full((n,), 1, dtype=torch.int64, device=dev)
        x1 = torch.full((n,), 3, dtype=torch.int64, device=dev)
        x0[n - 1] = -5
        z = torch.empty(1, dtype=torch.int64, device=dev)
        ws = torch.empty(ctx.scratch_bytes("aby3_sqnorm", 1), dtype=torch.uint8, device=dev)
        ctx.call("aby3_sqnorm_local", [x0], [x1], [n], 1, KEY01, 5, KEY01, 5, ws, z)
        assert z.item() == 7 * (n - 1) - 5
        y = torch.empty(n, dtype=torch.int64, device=dev)
        zero, four = torch.zeros(1, dtype=torch.int64, device=dev), torch.full((1,), 4 << 32, dtype=torch.int64, device=dev)
        x0 <<= 17
        ctx.call("aby3_clip_local", 0, [x0], [x1], [n], 1, zero, four, zero, 1 << 16, 16, 0, 0, y, torch.empty_like(zero))  # norm 2, bound 1
        assert y[0].item() == 1 << 16 and y[n - 2].item() == 1 << 16 and y[n - 1].item() == -5 << 16
        del x0, x1, y
        torch.cuda.empty_cache()


NORMS = [0, 1, 2, 3, (1 << 32) - 1, 1 << 32, (1 << 32) + 1, 123456789012345, (1 << 62) + 12345, (1 << 63) + 5, (1 << 64) - 1]


@pytest.mark.parametrize("number,max_norm", [(0, 0), (0, 1), (0, (1 << 62) - 1), (16, 1 << 16), (16, 0), (16, 12345), (16, (1 << 46) - 1),
                                             (31, 1), (31, (1 << 31) - 1), (7, 1000)])
def test_clip_factor(gpu, number, max_norm):
    """The factor for squared norms at and next to the bound, zero, and beyond 2^63."""
    edge = [(max_norm << k) ** 2 // q for k in (0, 1) for q in (1, 2, 3, 4)]
    for S in NORMS + [s for e in edge for s in (e - 1, e, e + 1) if 0 <= s < 2 ** 64]:
        z0, z1 = 0x9E3779B97F4A7C15, 0xC2B2AE3D27D4EB4F
        z = [np.array([v % 2 ** 64], np.uint64).view(np.int64) for v in (S - z0 - z1, z0, z1)]
        x = np.array([1 << 20, -(1 << 20), 7], np.int64)
        y, c = gpu.aby3_clip_local(0, [x], [x], *z, max_norm, number, KEY12, 0)
        want = ref.clip_factor(S, max_norm, number)
        assert int(c[0]) == want, (S, int(c[0]), want)
        assert np.array_equal(y, (x * want) >> number)


@pytest.mark.parametrize("lens", LENS, ids=lambda v: f"{len(v)}x{max(v)}")
@pytest.mark.parametrize("pop12", [0, 1, 12345])
def test_clip_segments(gpu, lens, pop12):
    rng = np.random.default_rng(sum(lens) + len(lens) + pop12)
    X0, X1 = [rnd(rng, n) for n in lens], [rnd(rng, n) for n in lens]
    S = 9 << 32  # norm 3, bound 1
    z = [np.array([v], np.int64) for v in (S, 5, -5)]
    c = ref.clip_factor(S, 1 << 16, 16)
    w = prg_pops(KEY12, pop12, max(sum(lens), 1))[:sum(lens)]
    x0, x1 = np.concatenate(X0), np.concatenate(X1)
    with np.errstate(over="ignore"):
        want = [(x0 * c) >> 16, (((x0 + x1) * c) >> 16) - w, w]
    for party in range(3):
        y, coef = gpu.aby3_clip_local(party, X0, X1, *z, 1 << 16, 16, KEY12, pop12)
        assert int(coef[0]) == c
        assert np.array_equal(y, want[party]), party


# ------------------------------------------------------------------ log probabilities of opened logits
def share(rng, x, shares):
    out = [rnd(rng, x.size) for _ in range(shares - 1)]
    first = ref.words(x.ravel()).copy()
    for s in out:
        first -= ref.words(s)
    return [first.view(np.int64)] + out + [None] * (3 - shares)


def logit_rows(kind, rng, rows, vocab, frac):
    unit = 2.0 ** frac
    if kind == "normal":
        return (rng.normal(size=(rows, vocab)) * 3 * unit).astype(np.int64)
    if kind == "ties":  # a handful of values, so that alternatives tie at the border
        return (rng.integers(-2, 3, (rows, vocab)) * unit).astype(np.int64)
    if kind == "peak":  # one token takes everything, the rest are masked to the lowest word
        x = np.full((rows, vocab), LOWEST, np.int64)
        x[np.arange(rows), rng.integers(0, vocab, rows)] = rng.integers(-5, 5, rows)
        return x
    if kind == "lowest":  # nothing is left: all of the row is masked
        return np.full((rows, vocab), LOWEST, np.int64)
    if kind == "extreme":
        return rng.choice(np.array([LOWEST, LOWEST + 1, 0, HIGHEST - 1, HIGHEST], np.int64), (rows, vocab))
    if kind == "rising":  # the maximum moves with every word
        return (np.arange(vocab, dtype=np.float64)[None, :] * unit * 0.01 + rng.normal(size=(rows, 1))).astype(np.int64)
    if kind == "falling":
        return (-np.arange(vocab, dtype=np.float64)[None, :] * unit * 0.01 + rng.normal(size=(rows, 1))).astype(np.int64)
    return rnd(rng, rows, vocab)  # "words"


def logprob_bounds(x, frac, want, vocab):
    """Half steps: a lane sums at most vocab / 64 terms one after the other and joins fewer than 64 partial sums; each term
    is off by its distance's rounding (distance e^-distance <= 0.37) and the exponential's (2 steps)."""
    logp, H, order, top_logp, m, ls = want
    terms = vocab / 64 + 64 + 4
    d_ls = terms * STEP + np.abs(ls) * 2 * STEP
    return d_ls, 2 * terms * STEP * (1 + np.abs(H)) + 4 * STEP * (np.abs(ls) + np.abs(H))


KINDS = ["normal", "ties", "peak", "lowest", "extreme", "rising", "falling", "words"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,vocab,per_row,top,shares", [(1, 1, 1, 1, 3), (3, 2, 2, 2, 1), (128, 10, 1, 3, 2), (5, 63, 1, 32, 3),
                                                           (9, 64, 0, 5, 2), (4, 257, 3, 0, 3), (3, 1009, 5, 20, 3),
                                                           (2, 32771, 1, 32, 3), (1, 131072, 2, 20, 3), (300, 515, 1, 5, 2),
                                                           (1, 200001, 1, 1, 1), (600, 64, 1, 32, 3)])
def test_logprobs(gpu, kind, rows, vocab, per_row, top, shares):
    rng = np.random.default_rng(rows * 7 + vocab + KINDS.index(kind))
    for frac in (16, 0, 40, 62) if kind in ("extreme", "words", "normal") and vocab < 2000 else (16,):
        x = logit_rows(kind, rng, rows, vocab, min(frac, 55))
        ids = rng.integers(0, vocab, (rows, per_row))
        bad = rng.random((rows, per_row)) < 0.1
        ids[bad] = rng.choice(np.array([-1, vocab, LOWEST, 2 ** 40], np.int64), int(bad.sum()))
        got = gpu.reveal_logprobs(*share(rng, x, shares), rows, vocab, frac, ids.ravel(), top)
        want = ref.logprobs(x, frac, ids, top)
        logp, H, top_ids, top_logp, m, ls = [g.reshape(w.shape) for g, w in zip(got, want)]
        assert np.array_equal(m, want[4])
        assert np.array_equal(top_ids, want[2])
        d_ls, d_H = logprob_bounds(x, frac, want, vocab)
        assert (np.abs(ls - want[5]) <= d_ls).all()
        assert (np.abs(H - want[1]) <= d_H).all()
        assert (np.abs(logp - want[0]) <= d_ls[:, None] + 3 * STEP * np.abs(want[0])).all()
        assert (np.abs(top_logp - want[3]) <= d_ls[:, None] + 3 * STEP * np.abs(want[3])).all()
        assert (logp[(ids < 0) | (ids >= vocab)] == 0).all()


@pytest.mark.parametrize("kind", ["normal", "ties", "peak", "lowest", "extreme"])
@pytest.mark.parametrize("rows,vocab,per_row,shares", [(1, 1, 1, 3), (3, 2, 2, 1), (128, 10, 1, 2), (5, 63, 1, 3), (9, 64, 0, 2),
                                                       (4, 257, 3, 3), (3, 1009, 70, 3), (2, 32771, 1, 3), (1, 131072, 2, 3),
                                                       (300, 515, 1, 2), (2, 300, 600, 3)])
@pytest.mark.parametrize("with_entropy", [False, True])
def test_logprobs_grad(gpu, kind, rows, vocab, per_row, shares, with_entropy):
    rng = np.random.default_rng(rows * 7 + vocab + KINDS.index(kind))
    frac, grad_frac = 16, 20
    x = logit_rows(kind, rng, rows, vocab, frac)
    ids = rng.integers(0, vocab, (rows, per_row))
    bad = rng.random((rows, per_row)) < 0.1
    ids[bad] = rng.choice(np.array([-1, vocab, LOWEST, 2 ** 40], np.int64), int(bad.sum()))
    f32 = np.float32
    _, H, _, _, m, ls = ref.logprobs(x, frac, ids, 0)
    H, ls = H.astype(f32), ls.astype(f32)
    d_logp, d_ent = rng.normal(size=(rows, per_row)).astype(f32), (rng.normal(size=rows).astype(f32) if with_entropy else None)
    grad, words = gpu.reveal_logprobs_grad(*share(rng, x, shares), rows, vocab, frac, ids.ravel(), d_logp.ravel(), d_ent, m, ls,
                                           H if with_entropy else None, grad_frac)
    want, err = ref.logprobs_grad(x, frac, ids, d_logp, d_ent, m, ls, H)
    grad = grad.reshape(rows, vocab)
    assert (np.abs(grad - want) <= err + 1e-37).all(), np.abs(grad - want).max()
    # the words are the floats, rounded once
    assert np.array_equal(words.reshape(rows, vocab), np.rint(grad.astype(np.float64) * 2.0 ** grad_frac).astype(np.int64))


def test_logprobs_grad_against_differences(gpu):
    """The gradient along random directions against central differences of the 64-bit loss."""
    rng = np.random.default_rng(12)
    rows, vocab, per_row, frac = 3, 50, 2, 40
    x = (rng.normal(size=(rows, vocab)) * 2.0 ** frac).astype(np.int64)
    ids = rng.integers(0, vocab, (rows, per_row))
    ids[0, 1] = ids[0, 0]  # the same token twice
    ids[1, 0] = -1
    w, h = rng.normal(size=(rows, per_row)).astype(np.float32), rng.normal(size=rows).astype(np.float32)
    _, H, _, _, m, ls = ref.logprobs(x, frac, ids, 0)
    grad, _ = gpu.reveal_logprobs_grad(x.ravel(), None, None, rows, vocab, frac, ids.ravel(), w.ravel(), h, m, ls.astype(np.float32),
                                       H.astype(np.float32), 20)
    grad = grad.reshape(rows, vocab).astype(np.float64)

    def loss(y):
        logp, ent = ref.logprobs(y, frac, ids, 0)[:2]
        return (logp * w).sum() + (ent * h).sum()

    eps = 2 ** 24  # 2^-16 in the logits: the quotient's own error is about eps^2 times the third derivative, below 1e-8
    for _ in range(20):
        d = rng.integers(-1, 2, (rows, vocab))
        quotient = (loss(x + eps * d) - loss(x - eps * d)) / (2 * eps * 2.0 ** -frac)
        assert abs(quotient - (grad * d).sum()) < 2e-5 * np.abs(grad).sum() + 1e-8


def test_logprobs_leave_out_what_is_not_asked_for(gpu):
    """NULL outputs: only row_max; only words of the gradient."""
    ctx = gpu.ctx
    rng = np.random.default_rng(1)
    rows, vocab = 6, 777
    x = logit_rows("normal", rng, rows, vocab, 16)
    dx = ctx.to_device(x.ravel())
    m, ls, words = ctx.empty(np.int64, rows), ctx.empty(np.float32, rows), ctx.empty(np.int64, rows * vocab)
    ws = ctx.empty(np.uint8, ctx.scratch_bytes("reveal_logprobs", rows, vocab, 0))
    ctx.call("reveal_logprobs", dx, None, None, rows, vocab, 16, None, 0, 0, ws, None, None, None, None, m, None)
    ctx.call("reveal_logprobs", dx, None, None, rows, vocab, 16, None, 0, 0, ws, None, None, None, None, None, ls)
    ids, w = ctx.to_device(np.arange(rows, dtype=np.int64)), ctx.to_device(np.ones(rows, np.float32))
    ctx.call("reveal_logprobs_grad", dx, None, None, rows, vocab, 16, ids, 1, w, None, m, ls, None, None, words, 30)
    ctx.sync()
    assert np.array_equal(m.to_host(), x.max(1))
    want, err = ref.logprobs_grad(x, 16, np.arange(rows)[:, None], np.ones((rows, 1), np.float32), None, x.max(1), ls.to_host(), None)
    assert (np.abs(words.to_host().reshape(rows, vocab) * 2.0 ** -30 - want) <= err + 2.0 ** -31).all()


def test_logprobs_grad_words_saturate(gpu):
    """Errors too large for a word end at the ends of the range."""
    x = np.zeros((2, 2), np.int64)
    ls = np.full(2, np.log(2), np.float32)
    w = np.array([[1e30], [-1e30]], np.float32)
    _, words = gpu.reveal_logprobs_grad(x.ravel(), None, None, 2, 2, 16, np.zeros(2, np.int64), w.ravel(), None, np.zeros(2, np.int64),
                                        ls, None, 62)
    assert words.tolist() == [HIGHEST, LOWEST, LOWEST, HIGHEST]


@pytest.mark.parametrize("rows,vocab", [((1 << 16) + 3, 65537), (3, (1 << 31) - 1)])
def test_logprobs_beyond_four_billion_words(resident, rows, vocab):
    ctx, torch, dev, be, side = resident
    with torch.cuda.stream(side):
        x = torch.zeros(rows * vocab, dtype=torch.int64, device=dev)
        last = rows - 1
        x[last * vocab + vocab - 2] = 40 << 16
        x[last * vocab] = 39 << 16
        ids = torch.full((rows,), vocab - 2, dtype=torch.int64, device=dev)
        f = lambda *s: torch.empty(*s, dtype=torch.float32, device=dev)
        logp, ent, ls, tl = f(rows), f(rows), f(rows), f(rows * 2)
        ti, m = torch.empty(rows * 2, dtype=torch.int64, device=dev), torch.empty(rows, dtype=torch.int64, device=dev)
        ws = torch.empty(ctx.scratch_bytes("reveal_logprobs", rows, vocab, 2), dtype=torch.uint8, device=dev)
        ctx.call("reveal_logprobs", x, None, None, rows, vocab, 16, ids, 1, 2, ws, logp, ent, ti, tl, m, ls)
        side.synchronize()
        uniform = np.log(vocab)
        bound = (vocab / 64 + 70) * STEP + 4 * STEP * uniform
        assert m[last].item() == 40 << 16 and m[0].item() == 0
        assert ti[-2:].tolist() == [vocab - 2, 0] and ti[:2].tolist() == [0, 1]
        assert abs(ent[0].item() - uniform) <= min(2 * bound * (1 + uniform), 1e-3) and abs(logp[0].item() + uniform) <= min(bound, 1e-3)
        assert abs(ls[last].item() - np.log1p(np.exp(-1.0) + (vocab - 2) * np.exp(-40.0))) <= 1e-6
        del x, ws
        torch.cuda.empty_cache()


def test_more_rows_than_one_launch_takes(resident):
    """Rows, table rows and tokens beyond what the grid of one launch holds."""
    ctx, torch, dev, be, side = resident
    i64 = lambda *s: torch.empty(*s, dtype=torch.int64, device=dev)
    with torch.cuda.stream(side):
        rows = (1 << 24) + 5
        x = torch.zeros(rows, 2, dtype=torch.int64, device=dev)
        x[-1, 1] = x[1 << 22, 1] = 1 << 16
        ids = torch.ones(rows, dtype=torch.int64, device=dev)
        f = lambda *s: torch.empty(*s, dtype=torch.float32, device=dev)
        logp, ent, ls, tl, ti, m = f(rows), f(rows), f(rows), f(rows), i64(rows), i64(rows)
        ws = torch.empty(ctx.scratch_bytes("reveal_logprobs", rows, 2, 1), dtype=torch.uint8, device=dev)
        ctx.call("reveal_logprobs", x, None, None, rows, 2, 16, ids, 1, 1, ws, logp, ent, ti, tl, m, ls)
        grad, w = f(rows, 2), torch.ones(rows, dtype=torch.float32, device=dev)
        ctx.call("reveal_logprobs_grad", x, None, None, rows, 2, 16, ids, 1, w, None, m, ls, None, grad, None, 0)
        peak = torch.tensor([1 << 22, rows - 1], device=dev)
        assert ti.nonzero()[:, 0].tolist() == peak.tolist() and m.nonzero()[:, 0].tolist() == peak.tolist()
        lp1 = -np.log1p(np.exp(-1.0))
        assert (logp[peak] - lp1).abs().max().item() < 8 * STEP
        even = torch.ones(rows, dtype=torch.bool, device=dev)
        even[peak] = False
        assert (logp[even] + np.log(2)).abs().max().item() < 8 * STEP and (ent[even] - np.log(2)).abs().max().item() < 16 * STEP
        assert (grad[even] - torch.tensor([-0.5, 0.5], device=dev)).abs().max().item() < 8 * STEP
        p = np.exp(lp1)
        assert (grad[peak] - torch.tensor([p - 1, 1 - p], device=dev, dtype=torch.float32)).abs().max().item() < 8 * STEP
        del x, ids, logp, ent, ls, tl, ti, m, grad, w, even
        torch.cuda.empty_cache()
        # lookup of many wide rows: one workgroup a row
        n, dim = (1 << 23) + 3, 300
        T = torch.arange(7 * dim, dtype=torch.int64, device=dev).view(7, dim)
        ids = torch.arange(n, device=dev) % 7
        E = i64(n, dim)
        ctx.call("ring_embed", T, None, 7, dim, ids, n, 1, 0, E, None)
        for a in range(0, n, 1 << 21):
            assert torch.equal(E[a:a + (1 << 21)], T[ids[a:a + (1 << 21)]])
        del E
        torch.cuda.empty_cache()
        # the gradient of a table of many rows
        vocab, dim, n = (1 << 23) + 9, 300, 40
        D, G = i64(vocab, dim), torch.arange(n * dim, dtype=torch.int64, device=dev).view(n, dim) + 1
        ids = torch.full((n,), vocab - 1, dtype=torch.int64, device=dev)
        ids[:3] = torch.tensor([0, 5 << 20, vocab - 2], device=dev)
        ws = torch.empty(ctx.scratch_bytes("ring_embed_grad", n, vocab, dim), dtype=torch.uint8, device=dev)
        D.fill_(-1)
        ctx.call("ring_embed_grad", G, None, ids, n, vocab, dim, 2, 0, 0, ws, D, None)
        for k in range(3):
            assert torch.equal(D[ids[k]], 2 * G[k])
        assert torch.equal(D[vocab - 1], 2 * G[3:].sum(0))
        D[ids] = 0
        assert not any(D[a:a + (1 << 20)].any().item() for a in range(0, vocab, 1 << 20))
        del D, ws
        torch.cuda.empty_cache()


# ------------------------------------------------------------------ together
def secure_step(be, w, E, W, ids, targets, rows, vocab, dim, frac):
    """One step of a private next-token model (table E, head W, both shared) on public text: lookup, product with the head,
    truncation, opened log probabilities, the error in ring words, the gradients of head and table, clipping."""
    Es, Ws = pr.aby3_share(w, E, vocab * dim), pr.aby3_share(w, W, dim * vocab)
    X = pr.aby3_embed(w, Es, vocab, dim, ids)
    L = pr.aby3_trunc(w, pr.aby3_matmul(w, X, Ws, rows, dim, vocab), frac)
    out = pr.aby3_reveal_logprobs(w, L, rows, vocab, frac, targets, top=3)
    weight = np.full(rows, -1.0 / rows, np.float32)  # the mean negative log probability
    weight = be.up(weight) if hasattr(be, "up") else weight
    tensors = []
    j0 = out[0]
    _, err = be.reveal_logprobs_grad(L[2][0], L[0][0], L[0][1], rows, vocab, frac, targets, weight, None, j0[4], j0[5], None, frac)
    return X, L, out, err


def test_a_private_models_training_step(gpu, orc):
    """Lookup -> head -> opened loss -> error -> gradients of both matrices -> global norm -> clip -> update, on three
    parties' shares; the opened result is the fixed-point computation in the clear, up to the truncations' last bit."""
    rng = np.random.default_rng(5)
    rows, vocab, dim, frac = 24, 301, 48, 16
    one = 1 << frac
    E = (rng.normal(size=(vocab, dim)) * one).astype(np.int64)
    W = (rng.normal(size=(dim, vocab)) * 0.3 * one).astype(np.int64)
    ids, targets = rng.integers(0, vocab, rows), rng.integers(0, vocab, rows)
    ids[3] = ids[4]
    w = pr.World(gpu)
    X, L, out, err = secure_step(gpu, w, E.ravel(), W.ravel(), ids, targets, rows, vocab, dim, frac)
    open3 = lambda S: (ref.words(S[0][0]) + ref.words(S[1][0]) + ref.words(S[2][0])).view(np.int64)
    assert np.array_equal(open3(X).reshape(rows, dim), E[ids])
    logits = open3(L).reshape(rows, vocab)
    assert np.abs(logits - ((E[ids] @ W) >> frac)).max() <= 2
    want = ref.logprobs(logits, frac, targets[:, None], 3)
    for o in out:  # every party forms the same
        assert np.array_equal(o[2].reshape(rows, 3), want[2])
        assert np.abs(o[0] - want[0][:, 0]).max() < 1e-4 and np.array_equal(o[0], out[0][0])
    err = err.reshape(rows, vocab)
    p = np.exp(-((want[4][:, None] - logits) * 2.0 ** -frac + want[5][:, None]))
    p[np.arange(rows), targets] -= 1
    assert np.abs(err * 2.0 ** -frac - p / rows).max() < 2e-5
    # gradients: share by public, each share on its own; then truncation back to frac bits
    Ws = [pr.aby3_share(pr.World(gpu, record=False), W.ravel(), W.size)[j] for j in range(3)]
    dW = [tuple(gpu.ring_gemm(x, err.ravel(), dim, rows, vocab, layA=1) for x in X[j]) for j in range(3)]
    dX = [tuple(gpu.ring_gemm(err.ravel(), s, rows, vocab, dim, layB=1) for s in Ws[j]) for j in range(3)]
    assert np.array_equal(open3(dW).reshape(dim, vocab), E[ids].T @ err)
    assert np.array_equal(open3(dX).reshape(rows, dim), err @ W.T)
    dW, dX = pr.aby3_trunc(w, dW, frac), pr.aby3_trunc(w, dX, frac)
    dE = pr.aby3_embed_grad(w, dX, ids, vocab, dim)
    plain = np.zeros((vocab, dim), np.int64)
    np.add.at(plain, ids, open3(dX).reshape(rows, dim))
    assert np.array_equal(open3(dE).reshape(vocab, dim), plain)
    # clip to a tenth of the norm
    grads = np.concatenate([plain.ravel(), open3(dW)])
    S = int(sum(int(v) * int(v) for v in grads))
    max_norm = int(np.sqrt(S) / 10)
    clipped, coef = pr.aby3_clip(w, [dE, dW], max_norm, frac)
    z = [e for t, e in w.log if t.startswith("sqnorm")]
    assert (int(z[0][0]) + int(z[1][0]) + int(z[2][0])) % 2 ** 64 == S
    c = ref.clip_factor(S, max_norm, frac)
    assert int(coef[0]) == c
    got = open3(clipped)
    assert np.abs(got - ((grads * c) >> frac)).max() <= 2
    assert np.sqrt((got.astype(np.float64) ** 2).sum()) <= max_norm * 1.01 + 2 * np.sqrt(got.size)


def test_the_step_on_device_arrays_gives_the_same_words(gpu, resident):
    ctx, torch, dev, be, side = resident
    rng = np.random.default_rng(6)
    rows, vocab, dim, frac = 7, 130, 33, 16
    E, W = [(rng.normal(size=vocab * dim) * (1 << frac)).astype(np.int64) for _ in range(2)]
    ids, targets = rng.integers(0, vocab, rows), rng.integers(0, vocab, rows)
    a = secure_step(gpu, pr.World(gpu), E, W, ids, targets, rows, vocab, dim, frac)
    with torch.cuda.stream(side):
        b = secure_step(be, pr.World(be, record=False), be.up(E), be.up(W), be.up(ids), be.up(targets), rows, vocab, dim, frac)
        assert np.array_equal(be.down(b[3]), a[3])
        for j in range(3):
            assert np.array_equal(be.down(b[1][j][0]), a[1][j][0])
            for u, v in zip(b[2][j], a[2][j]):
                assert np.array_equal(be.down(u), v)


# ------------------------------------------------------------------ graphs and streams
def test_operators_replayed_from_graphs(resident):
    """Everything captured once and replayed on new inputs, with eager work between the replays, equals the eager calls."""
    ctx, torch, dev, be, side = resident
    rng = np.random.default_rng(9)
    vocab, dim, n, rows = 997, 130, 600, 40
    lens = [1000, 1, 33333]
    i64 = lambda *s: torch.empty(*s, dtype=torch.int64, device=dev)
    f32 = lambda *s: torch.empty(*s, dtype=torch.float32, device=dev)
    fill = lambda t: t.copy_(torch.from_numpy(rnd(rng, *t.shape)))
    with torch.cuda.stream(side):
        T0, T1, G0, G1 = i64(vocab, dim), i64(vocab, dim), i64(n, dim), i64(n, dim)
        ids = i64(n)
        E0, E1, D0, D1 = i64(n, dim), i64(n, dim), i64(vocab, dim), i64(vocab, dim)
        X0, X1 = [i64(k) for k in lens], [i64(k) for k in lens]
        z, zero, y, coef = i64(1), torch.zeros(1, dtype=torch.int64, device=dev), i64(sum(lens)), i64(1)
        y1 = i64(sum(lens))
        x = i64(rows, vocab)
        tgt = i64(rows, 2)
        outs = [f32(rows, 2), f32(rows), i64(rows, 5), f32(rows, 5), i64(rows), f32(rows)]
        w = torch.full((rows, 2), 0.5, device=dev)
        grad, words = f32(rows, vocab), i64(rows, vocab)
        sc = lambda name, *s: torch.empty(ctx.scratch_bytes(name, *s), dtype=torch.uint8, device=dev)
        s1, s2, s3 = sc("ring_embed_grad", n, vocab, dim), sc("aby3_sqnorm", 3), sc("reveal_logprobs", rows, vocab, 5)

    def calls():
        ctx.call("ring_embed", T0, T1, vocab, dim, ids, n, 5, 0, E0, E1)
        ctx.call("ring_embed_grad", G0, G1, ids, n, vocab, dim, 5, 0, 0, s1, D0, D1)
        ctx.call("aby3_sqnorm_local", X0, X1, lens, 3, KEY01, 9, KEY20, 9, s2, z)
        ctx.call("aby3_clip_local", 0, X0, X1, lens, 3, z, zero, zero, 1 << 16, 16, 0, 0, y, coef)
        ctx.call("aby3_clip_local", 1, X0, X1, lens, 3, z, zero, zero, 1 << 16, 16, KEY12, 77, y1, coef)
        ctx.call("reveal_logprobs", x, None, None, rows, vocab, 16, tgt, 2, 5, s3, *outs)
        ctx.call("reveal_logprobs_grad", x, None, None, rows, vocab, 16, tgt, 2, w, None, outs[4], outs[5], None, grad, words, 24)

    results = [E0, E1, D0, D1, z, y, y1, coef, *outs, grad, words]

    def refill():
        for t in (T0, T1, G0, G1, *X0, *X1):
            fill(t)
        ids.copy_(torch.from_numpy(tokens(rng, n, vocab)))
        x.copy_(torch.from_numpy(logit_rows("normal", rng, rows, vocab, 16)))
        tgt.copy_(torch.from_numpy(rng.integers(-1, vocab, (rows, 2))))

    with torch.cuda.stream(side):
        refill()
        calls()
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side, capture_error_mode="thread_local"):
        calls()
    for _ in range(4):
        with torch.cuda.stream(side):
            refill()
            calls()
            want = [t.clone() for t in results]
            for t in results:
                t.zero_()
            side.synchronize()
            g.replay()
            side.synchronize()
            for k, (a, b) in enumerate(zip(results, want)):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), k


def test_two_contexts_at_once(resident):
    """Two contexts on two streams of one GPU, each with its own scratch, give what each gives alone."""
    ctx, torch, dev, be, side = resident
    from mpc_amd import Context
    other = Context(0)
    s2 = torch.cuda.Stream(dev)
    other.call("set_stream", s2.cuda_stream)
    rng = np.random.default_rng(4)
    vocab, dim, n = 700, 257, 20000
    jobs = []
    for c, s in ((ctx, side), (other, s2)):
        with torch.cuda.stream(s):
            G = torch.from_numpy(rnd(rng, n, dim)).to(dev)
            ids = torch.from_numpy(tokens(rng, n, vocab)).to(dev)
            D = torch.empty(vocab, dim, dtype=torch.int64, device=dev)
            x = torch.from_numpy(logit_rows("normal", rng, 3, 100003, 16)).to(dev)
            m, ls = torch.empty(3, dtype=torch.int64, device=dev), torch.empty(3, dtype=torch.float32, device=dev)
            sc = lambda name, *a: torch.empty(c.scratch_bytes(name, *a), dtype=torch.uint8, device=dev)
            jobs.append((c, s, G, ids, D, x, m, ls, sc("ring_embed_grad", n, vocab, dim), sc("reveal_logprobs", 3, 100003, 0)))
    torch.cuda.synchronize()
    for _ in range(20):
        for c, s, G, ids, D, x, m, ls, w1, w2 in jobs:
            c.call("ring_embed_grad", G, None, ids, n, vocab, dim, 1, 0, 0, w1, D, None)
            c.call("reveal_logprobs", x, None, None, 3, 100003, 16, None, 0, 0, w2, None, None, None, None, m, ls)
    torch.cuda.synchronize()
    for c, s, G, ids, D, x, m, ls, w1, w2 in jobs:
        assert np.array_equal(D.cpu().numpy().ravel(), ref.embed_grad(G.cpu().numpy().ravel(), ids.cpu().numpy(), vocab, dim, 1, 0))
        assert torch.equal(m, x.amax(1))
        want = ref.logprobs(x.cpu().numpy(), 16, np.zeros((3, 0), np.int64), 0)[5]
        assert np.abs(ls.cpu().numpy() - want).max() < (100003 / 64 + 70) * STEP + 4 * STEP * np.abs(want).max()
    other.close()


@pytest.mark.parametrize("lens", [[(1 << 23) - 1, 5, 1 << 23, 0, 1, (1 << 23) + 4097, 300, 0], [4096] * 20 + [1] * 70 + [64, 4095, 0, 8192] * 30,
                                  [17, 47, 63, 65, 1, 4031] * 40], ids=["long", "aligned", "odd"])
def test_clip_of_tensors_that_begin_and_end_anywhere(gpu, lens):
    """Party 1 finds the tensor of a word per wavefront of 4096 words, or per visit of 64."""
    rng = np.random.default_rng(77)
    X0, X1 = [rnd(rng, n) for n in lens], [rnd(rng, n) for n in lens]
    z = [np.array([v], np.int64) for v in (25 << 32, 0, 0)]
    c = ref.clip_factor(25 << 32, 1 << 16, 16)
    w = prg_pops(KEY12, 9, sum(lens))
    with np.errstate(over="ignore"):
        want = ((((np.concatenate(X0) + np.concatenate(X1)) * c) >> 16) - w)
    y, coef = gpu.aby3_clip_local(1, X0, X1, *z, 1 << 16, 16, KEY12, 9)
    assert int(coef[0]) == c and np.array_equal(y, want)
