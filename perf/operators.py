"""Cases of the language-model operators on secret shares, and their plain forms in elementary torch operations.

A shared word is an int64 mod 2^64; an ABY3 party holds two of the three shares of every value (replicated), a SecureNN /
MyEngine party one of two (additive).  Reals are fixed point with FRAC fractional bits.  Text (token ids) is public, what
the model has learnt is shared:

  embed         E_k[t] = (scale * T_k[ids[t]]) >> shift                   rows of a shared table
  embed_grad    dT_k[v] = (scale * sum_{t: ids[t] = v} G_k[t]) >> shift   the whole (dense) gradient of the table
  norm          z = sum x0 (x0 + 2 x1) + mask_next - mask_prev            a party's share of the squared global norm
  clip          y = (c x0) >> FRAC, c = max {c <= 2^FRAC: c^2 S <= (M 2^FRAC)^2}, S the opened squared norm
  logprobs      log probabilities of given tokens, entropy and the top alternatives of opened logits
  logprobs_grad the gradient of (weighted log probabilities + weighted entropy) with respect to the logits
"""
import functools
import math
import random

import numpy as np
import torch

own = False

FRAC = 16
SEED_NEXT, SEED_PREV = 0xAB01, 0xCA20  # party 0's generators: the streams it shares with parties 1 and 2
I64 = torch.int64
LO, HI = -2 ** 63, 2 ** 63 - 1


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one generated token: its row out of an ABY3 table, latency alone
        {"name": "embed_one_token", "op": "embed", "vocab": 32768, "dim": 256, "n": 1, "shares": 2, "scale": 16, "shift": 0},
        # a long batch of prompts against a wide table, scaled by sqrt(dim)
        {"name": "embed_prompts", "op": "embed", "vocab": 131072, "dim": 4096, "n": 16384, "shares": 2, "scale": 64,
         "shift": 0},
        # a short step of a small odd-sized table on one additive share (SecureNN), the fixed-point scale (2^FRAC
        # sqrt(dim)) taken back locally: launches count
        {"name": "embed_grad_small", "op": "embed_grad", "vocab": 1009, "dim": 129, "n": 999, "shares": 1, "scale": 744345,
         "shift": FRAC},
        # a training step of a large shared table: Zipf tokens, the dense gradient is most of the traffic
        {"name": "embed_grad_step", "op": "embed_grad", "vocab": 65536, "dim": 1024, "n": 65536, "shares": 2, "scale": 32,
         "shift": 0},
        # the gradients of the 784-128-128-10 MLP with biases
        {"name": "norm_mlp", "op": "norm", "tensors": 6, "total": 118282, "spread": 0},
        # a model of many tensors from a few words to tens of millions
        {"name": "norm_many", "op": "norm", "tensors": 293, "total": 200000003, "spread": 1},
        # clipping the same two sets
        {"name": "clip_mlp", "op": "clip", "tensors": 6, "total": 118282, "spread": 0},
        {"name": "clip_many", "op": "clip", "tensors": 293, "total": 200000003, "spread": 1},
        # one decoded token over a large vocabulary with its alternatives
        {"name": "logprobs_decode", "op": "logprobs", "rows": 1, "vocab": 131072, "shares": 3, "per_row": 1, "top": 20},
        # scoring a batch of text
        {"name": "logprobs_score", "op": "logprobs", "rows": 4096, "vocab": 32771, "shares": 3, "per_row": 1, "top": 5},
        # the error of the MLP's ten classes on its batch, opened from two additive shares
        {"name": "logprobs_grad_mlp", "op": "logprobs_grad", "rows": 128, "vocab": 10, "shares": 2, "per_row": 1},
        # the error of a training batch
        {"name": "logprobs_grad_step", "op": "logprobs_grad", "rows": 2048, "vocab": 32768, "shares": 3, "per_row": 1},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    op = rng.choice(["embed", "embed_grad", "norm", "clip", "logprobs", "logprobs_grad"])
    if op in ("embed", "embed_grad"):
        dim = _log_int(rng, 64, 4096)
        vocab = min(_log_int(rng, 500, 131072), (2 ** 26 if op == "embed_grad" else 2 ** 29) // dim)
        n = min(_log_int(rng, 1, 65536), 2 ** 26 // dim)
        shares = rng.choice([1, 2])
        return {"op": op, "vocab": vocab, "dim": dim, "n": n, "shares": shares,
                "scale": int(round(math.sqrt(dim) * (1 if shares == 2 else 2 ** FRAC))), "shift": FRAC if shares == 1 else 0}
    if op in ("norm", "clip"):
        tensors = _log_int(rng, 1, 400)
        return {"op": op, "tensors": tensors, "total": max(_log_int(rng, 1000, 150000000), tensors), "spread": rng.choice([0, 1])}
    vocab = _log_int(rng, 10, 200000)
    rows = min(_log_int(rng, 1, 8192), max(1, 2 ** 26 // vocab))
    case = {"op": op, "rows": rows, "vocab": vocab, "shares": rng.choice([1, 2, 3]), "per_row": rng.choice([1, 1, 2, 5])}
    if op == "logprobs":
        case["top"] = min(vocab, rng.choice([0, 1, 5, 20, 32]))
    return case


# ------------------------------------------------------------------ inputs
@functools.lru_cache(maxsize=None)
def _mask_word(seed, pop):
    """Word `pop` of the pop stream of a prvhash generator: five warm-up words, 320000 words of buffers, then the pops."""
    full = (1 << 64) - 1
    lcg = hsh = out = 0
    for _ in range(5 + 320000 + pop + 1):
        seed = seed * (lcg * 2 + 1) & full
        rs = (seed >> 32 | seed << 32) & full
        hsh = (hsh + rs + 0xAAAAAAAAAAAAAAAA) & full
        lcg = (lcg + seed + 0x5555555555555555) & full
        seed ^= hsh
        out = lcg ^ rs
    return _signed(out)


def _signed(w):
    w &= (1 << 64) - 1
    return w - (1 << 64) if w >> 63 else w


def _lengths(case):
    """How the words are spread over the tensors: the MLP's own sizes, equal parts, or sizes from a few words upwards."""
    k, total = case["tensors"], case["total"]
    if k == 6 and total == 118282:
        return [784 * 128, 128, 128 * 128, 128, 128 * 10, 10]
    weights = [(i % 7 + 1) ** 6 if case["spread"] else 1 for i in range(k)]
    lens = [max(1, total * w // sum(weights)) for w in weights]
    lens[-1] = max(1, lens[-1] + total - sum(lens))
    return lens


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 13)
    return g


def _words(g, *shape):
    return torch.randint(LO, HI, shape, dtype=I64, device="cuda", generator=g)


def _tokens(g, n, vocab):
    """Token ids with Zipf frequencies over a shuffled vocabulary; one in 64 is padding (-1)."""
    u = torch.rand(n, device="cuda", generator=g, dtype=torch.float64)
    rank = torch.exp(u * math.log(vocab)).to(I64).clamp_(1, vocab) - 1
    step = next(p for p in (7919, 104729, 1299709, 15485863) if math.gcd(p, vocab) == 1)
    ids = rank * step % vocab
    pad = torch.rand(n, device="cuda", generator=g) < 1 / 64
    return torch.where(pad & (torch.arange(n, device="cuda") > 0), torch.full_like(ids, -1), ids)


def prepare(case, seed):
    g = _gen(seed)
    st = dict(case)
    op = case["op"]
    if op in ("embed", "embed_grad"):
        v, d, n, k = case["vocab"], case["dim"], case["n"], case["shares"]
        st["ids"] = _tokens(g, n, v)
        src, dst = (v, n) if op == "embed" else (n, v)
        st["x"] = [_words(g, src, d) for _ in range(k)]
        st["out"] = [torch.empty(dst, d, dtype=I64, device="cuda") for _ in range(k)]
    elif op in ("norm", "clip"):
        lens = _lengths(case)
        st["x0"] = [_words(g, n) for n in lens]
        st["x1"] = [_words(g, n) for n in lens]
        if op == "norm":
            st["pop"] = int(seed) % 1000
            st["mask"] = [_mask_word(SEED_NEXT, st["pop"]), _mask_word(SEED_PREV, st["pop"])]
            st["z"] = torch.empty(1, dtype=I64, device="cuda")
        else:
            # the three shares of the squared norm, 2 FRAC fractional bits; norms around and above the bound
            rng = random.Random(int(seed))
            norm = math.exp(rng.uniform(math.log(0.5), math.log(100.0)))
            s = int(norm * norm * 2 ** (2 * FRAC))
            z0, z1 = rng.getrandbits(64), rng.getrandbits(64)
            st["z"] = [torch.tensor([_signed(w)], dtype=I64, device="cuda") for w in (s - z0 - z1, z0, z1)]
            st["max_norm"] = 2 ** FRAC
            st["y"] = torch.empty(sum(lens), dtype=I64, device="cuda")  # the message: the tensors one after the other
            st["coef"] = torch.empty(1, dtype=I64, device="cuda")
    else:
        r, v, k = case["rows"], case["vocab"], case["shares"]
        logits = (torch.randn(r, v, device="cuda", generator=g) * 3 * 2 ** FRAC).to(I64)
        shares = [_words(g, r, v) for _ in range(k - 1)]
        for s in shares:
            logits -= s
        st["shares_of"] = [logits] + shares
        ids = torch.randint(0, v, (r, case["per_row"]), dtype=I64, device="cuda", generator=g)
        pad = torch.rand(r, case["per_row"], device="cuda", generator=g) < 1 / 64
        st["ids"] = torch.where(pad, torch.full_like(ids, -1), ids)
        f32 = dict(dtype=torch.float32, device="cuda")
        if op == "logprobs":
            st["out"] = [torch.empty(r, case["per_row"], **f32), torch.empty(r, **f32),
                         torch.empty(r, case["top"], dtype=I64, device="cuda"), torch.empty(r, case["top"], **f32),
                         torch.empty(r, dtype=I64, device="cuda"), torch.empty(r, **f32)]
        else:
            # what the forward pass has left: the largest logit, the logarithm of the sum, the entropy of each row
            x = sum(st["shares_of"])
            st["row_max"] = x.amax(1)
            st["log_sum"], st["entropy"] = torch.empty(r, **f32), torch.empty(r, **f32)
            for i in range(0, r, 256):
                dist = (st["row_max"][i:i + 256, None] - x[i:i + 256]).double() / 2 ** FRAC
                e = torch.exp(-dist)
                tot = e.sum(1)
                st["log_sum"][i:i + 256] = tot.log().float()
                st["entropy"][i:i + 256] = (tot.log() + (dist * e).sum(1) / tot).float()
            st["d_logp"] = torch.randn(r, case["per_row"], generator=g, **f32) / r
            st["d_entropy"] = torch.randn(r, generator=g, **f32) * (0.01 / r)
            st["grad"] = torch.empty(r, v, **f32)
    return st


# ------------------------------------------------------------------ one pass
@functools.lru_cache(maxsize=None)
def _context():
    from mpc_amd import Context
    ctx = Context(torch.cuda.current_device())
    ctx.call("set_stream", torch.cuda.current_stream().cuda_stream)
    return ctx


def _scratch(st, name, *sizes):
    """The scratch memory that a caller keeps for an entry point."""
    if "scratch" not in st:
        st["scratch"] = torch.empty(_context().scratch_bytes(name, *sizes), dtype=torch.uint8, device="cuda")
    return st["scratch"]


def _pair(ts):
    return ts[0], (ts[1] if len(ts) > 1 else None)


def _three(ts):
    return ts[0], (ts[1] if len(ts) > 1 else None), (ts[2] if len(ts) > 2 else None)


def run(st):
    return (_run_own if own else _run_plain)[st["op"]](st)


def _own_embed(st):
    (t0, t1), (e0, e1) = _pair(st["x"]), _pair(st["out"])
    _context().call("ring_embed", t0, t1, st["vocab"], st["dim"], st["ids"], st["n"], st["scale"], st["shift"], e0, e1)
    return st["out"]


def _plain_embed(st):
    here = st["ids"] >= 0
    rows = st["ids"].clamp(min=0)
    keep = here.to(I64)[:, None] * st["scale"]
    return [(x[rows] * keep) >> st["shift"] for x in st["x"]]


def _own_embed_grad(st):
    (g0, g1), (d0, d1) = _pair(st["x"]), _pair(st["out"])
    ws = _scratch(st, "ring_embed_grad", st["n"], st["vocab"], st["dim"])
    _context().call("ring_embed_grad", g0, g1, st["ids"], st["n"], st["vocab"], st["dim"], st["scale"], st["shift"], 0, ws, d0, d1)
    return st["out"]


def _plain_embed_grad(st):
    keep = (st["ids"] >= 0).to(I64)[:, None]
    rows = st["ids"].clamp(min=0)
    return [(torch.zeros(st["vocab"], st["dim"], dtype=I64, device="cuda").index_add_(0, rows, x * keep) * st["scale"]) >> st["shift"]
            for x in st["x"]]


def _own_norm(st):
    ns = [t.numel() for t in st["x0"]]
    ws = _scratch(st, "aby3_sqnorm", len(ns))
    _context().call("aby3_sqnorm_local", st["x0"], st["x1"], ns, len(ns), SEED_NEXT, st["pop"], SEED_PREV, st["pop"], ws, st["z"])
    return st["z"]


def _plain_norm(st):
    z = sum((a * (a + 2 * b)).sum() for a, b in zip(st["x0"], st["x1"]))
    return (z + st["mask"][0] - st["mask"][1]).reshape(1)


def _own_clip(st):
    ns = [t.numel() for t in st["x0"]]
    z = st["z"]
    _context().call("aby3_clip_local", 0, st["x0"], st["x1"], ns, len(ns), z[0], z[1], z[2], st["max_norm"], FRAC, 0, 0, st["y"],
                    st["coef"])
    return [st["y"], st["coef"]]


def _plain_clip(st):
    s = (st["z"][0] + st["z"][1] + st["z"][2]).double()
    c = torch.floor(st["max_norm"] * 2.0 ** FRAC / torch.sqrt(s)).clamp(max=2.0 ** FRAC).to(I64)
    return [torch.cat([(x * c) >> FRAC for x in st["x0"]]), c]


def _own_logprobs(st):
    logp, ent, top_ids, top_logp, row_max, log_sum = st["out"]
    ws = _scratch(st, "reveal_logprobs", st["rows"], st["vocab"], st["top"])
    _context().call("reveal_logprobs", *_three(st["shares_of"]), st["rows"], st["vocab"], FRAC, st["ids"], st["per_row"],
                    st["top"], ws, logp, ent, top_ids, top_logp, row_max, log_sum)
    return st["out"]


def _plain_logprobs(st):
    x = sum(st["shares_of"])
    v = st["vocab"]
    row_max = x.amax(1)
    dist = (row_max[:, None] - x).float() / 2 ** FRAC
    e = torch.exp(-dist)
    tot = e.sum(1)
    log_sum = torch.log(tot)
    ent = log_sum + (dist * e).sum(1) / tot
    at = torch.gather(dist, 1, st["ids"].clamp(min=0))
    logp = torch.where(st["ids"] >= 0, -(at + log_sum[:, None]), torch.zeros_like(at))
    # keys that are all different: equal logits rank by the lower id
    key = x * 2 ** 18 + (v - 1 - torch.arange(v, device="cuda"))
    top = torch.topk(key, st["top"], 1).values
    top_ids = v - 1 - (top & (2 ** 18 - 1))
    top_logp = -(torch.gather(dist, 1, top_ids) + log_sum[:, None])
    return [logp, ent, top_ids, top_logp, row_max, log_sum]


def _own_logprobs_grad(st):
    _context().call("reveal_logprobs_grad", *_three(st["shares_of"]), st["rows"], st["vocab"], FRAC, st["ids"], st["per_row"],
                    st["d_logp"], st["d_entropy"], st["row_max"], st["log_sum"], st["entropy"], st["grad"], None, 0)
    return st["grad"]


def _plain_logprobs_grad(st):
    x = sum(st["shares_of"])
    dist = (st["row_max"][:, None] - x).float() / 2 ** FRAC
    logp = -(dist + st["log_sum"][:, None])
    p = torch.exp(logp)
    w = st["d_logp"] * (st["ids"] >= 0)
    grad = -p * w.sum(1, keepdim=True) - st["d_entropy"][:, None] * p * (logp + st["entropy"][:, None])
    return grad.scatter_add_(1, st["ids"].clamp(min=0), w)


_run_own = {"embed": _own_embed, "embed_grad": _own_embed_grad, "norm": _own_norm, "clip": _own_clip,
            "logprobs": _own_logprobs, "logprobs_grad": _own_logprobs_grad}
_run_plain = {"embed": _plain_embed, "embed_grad": _plain_embed_grad, "norm": _plain_norm, "clip": _plain_clip,
              "logprobs": _plain_logprobs, "logprobs_grad": _plain_logprobs_grad}


# ------------------------------------------------------------------ what a pass cannot do without
def _distinct(n, vocab):
    """How many table rows n tokens of _tokens touch, on average: each of them is read once."""
    r = np.arange(1, vocab)
    p = np.log1p(1 / r) / math.log(vocab) * (63 / 64)
    return max(1, int(np.sum(-np.expm1(n * np.log1p(-np.minimum(p, 1 - 1e-12))))))


def work(case):
    op = case["op"]
    if op in ("embed", "embed_grad"):
        v, d, n, k = case["vocab"], case["dim"], case["n"], case["shares"]
        if op == "embed":
            return {"bytes": 8 * k * d * (_distinct(n, v) + n) + 8 * n, "flops": k * d * n}
        return {"bytes": 8 * k * d * (n + v) + 8 * n, "flops": k * d * (n + v)}
    if op in ("norm", "clip"):
        n = sum(_lengths(case))
        return {"bytes": 16 * n + (8 if op == "norm" else 32), "flops": (3 if op == "norm" else 2) * n}
    r, v, k = case["rows"], case["vocab"], case["shares"]
    if op == "logprobs":
        return {"bytes": 8 * k * r * v + 8 * r * case["per_row"] + r * (4 * case["per_row"] + 16 + 12 * case["top"]),
                "flops": (k + 8) * r * v}
    return {"bytes": (8 * k + 4) * r * v + r * (12 * case["per_row"] + 20), "flops": (k + 8) * r * v}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "embed":
        out = []
        for x in st["x"]:
            e = torch.zeros(case["n"], case["dim"], dtype=I64, device="cuda")
            live = torch.nonzero(st["ids"] >= 0)[:, 0]
            e[live] = torch.bitwise_right_shift(torch.index_select(x, 0, st["ids"][live]) * case["scale"], case["shift"])
            out.append(e)
        return out
    if op == "embed_grad":
        # running sums over the tokens in the order of their ids; a row is the difference at its two ends
        order = torch.argsort(st["ids"], stable=True)
        ids = st["ids"][order]
        first = torch.searchsorted(ids, torch.arange(case["vocab"], device="cuda"))
        last = torch.searchsorted(ids, torch.arange(case["vocab"], device="cuda"), right=True)
        out = []
        for x in st["x"]:
            run_sum = torch.zeros(case["n"] + 1, case["dim"], dtype=I64, device="cuda")
            torch.cumsum(x[order], 0, out=run_sum[1:])
            out.append(((run_sum[last] - run_sum[first]) * case["scale"]) >> case["shift"])
        return out
    if op == "norm":
        if case["total"] > 20000000:
            return None
        a = np.concatenate([t.cpu().numpy() for t in st["x0"]]).view(np.uint64)
        b = np.concatenate([t.cpu().numpy() for t in st["x1"]]).view(np.uint64)
        z = int(np.dot(a, a)) + 2 * int(np.dot(a, b)) + st["mask"][0] - st["mask"][1]
        return torch.tensor([_signed(z)], dtype=I64, device="cuda")
    if op == "clip":
        s = sum(int(t.item()) for t in st["z"]) % 2 ** 64
        c = min(2 ** FRAC, math.isqrt((st["max_norm"] << FRAC) ** 2 // s)) if s else 2 ** FRAC
        return [torch.bitwise_right_shift(c * torch.cat(st["x0"]), FRAC), torch.tensor([c], dtype=I64, device="cuda")]
    rows = max(1, 2 ** 25 // case["vocab"])
    parts = [_exact_rows(st, case, slice(i, i + rows)) for i in range(0, case["rows"], rows)]
    if op == "logprobs":
        return [torch.cat(p) for p in zip(*parts)]
    return torch.cat(parts)


def _exact_rows(st, case, at):
    word = functools.reduce(torch.add, [s[at] for s in st["shares_of"]])
    ids, live = st["ids"][at].clamp(min=0), st["ids"][at] >= 0
    top_word = word.amax(1, keepdim=True)
    away = (word - top_word).double() * 2.0 ** -FRAC  # exact: the difference of two words
    log_sum = torch.logsumexp(away, 1, keepdim=True)
    logp = away - log_sum
    p = logp.exp()
    ent = -(p * logp).sum(1)
    if case["op"] == "logprobs":
        best, order = torch.sort(word, dim=1, descending=True, stable=True)
        order = order[:, :case["top"]]
        return [torch.where(live, logp.gather(1, ids), 0.0), ent, order, logp.gather(1, order), top_word[:, 0], log_sum[:, 0]]
    w = torch.where(live, st["d_logp"][at].double(), 0.0)
    grad = torch.zeros_like(p).scatter_add_(1, ids, w)
    grad -= p * w.sum(1, keepdim=True)
    return grad - st["d_entropy"][at].double()[:, None] * p * (logp + ent[:, None])
