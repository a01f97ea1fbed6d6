"""Cases of the decode operators that carry several hypotheses a sequence: beam selection,
the reorder of the beams' states, attention of a drafted token tree over a key/value cache,
and the acceptance of the tree's tokens.

``listed()`` and ``draw(rng)`` give cases, ``prepare(case, seed)`` the inputs a program has
in hand, ``run(state)`` one pass: in elementary torch operations where ``own`` is false,
through tabby_b200's entry points where it is true. ``exact`` evaluates the definitions in
64 bits, one sequence (or beam, or node) at a time.
"""
import math

import numpy as np
import torch

own = False

DEVICE = torch.device("cuda" if torch.cuda.is_available() else "cpu")
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2, "i32": 4}


# -- the cases ---------------------------------------------------------------------------
def _beam(name, batch, beams, vocab, n_out, dtype, pad=0, allowed=1.0):
    return {"name": name, "op": "beam", "batch": batch, "beams": beams, "vocab": vocab,
            "n_out": n_out, "dtype": dtype, "pad": pad, "allowed": allowed}


def _reorder(name, layers, batch, beams, heads, entries, dim, dtype, shortest, token_major):
    return {"name": name, "op": "reorder", "layers": layers, "batch": batch, "beams": beams,
            "heads": heads, "entries": entries, "dim": dim, "dtype": dtype,
            "shortest": shortest, "token_major": token_major}


def _tree(name, batch, nodes, heads, kv_heads, dim, longest, shortest, dtype, token_major):
    return {"name": name, "op": "tree", "batch": batch, "nodes": nodes, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "longest": longest, "shortest": shortest,
            "dtype": dtype, "token_major": token_major}


def _accept(name, layers, batch, nodes, depth, heads, entries, dim, dtype):
    return {"name": name, "op": "accept", "layers": layers, "batch": batch, "nodes": nodes,
            "depth": depth, "heads": heads, "entries": entries, "dim": dim, "dtype": dtype}


def listed():
    return [
        # One prompt searched with four beams: the smallest selection, bound by latency.
        _beam("beam one prompt", 1, 4, 151936, 8, "f32"),
        # A served batch of 32 prompts, 8 beams each, the logits as the LM head leaves them.
        _beam("beam served batch", 32, 8, 151936, 16, "f32"),
        # Half-precision logits of an odd vocabulary: every other row starts off alignment.
        _beam("beam odd vocabulary", 12, 5, 50257, 10, "bf16"),
        # Wide beams under a grammar that bans most tokens (-inf), padded rows.
        _beam("beam wide constrained", 4, 32, 49152, 64, "f16", pad=64, allowed=0.02),
        # The caches of one prompt's beams right after a short prompt (24 layers, K and V).
        _reorder("reorder one prompt", 48, 1, 4, 2, 256, 64, "bf16", 40, False),
        # The caches of a served batch, head-major, ragged lengths.
        _reorder("reorder served batch", 16, 16, 4, 8, 2048, 128, "bf16", 256, False),
        # Token-major caches of odd sizes in fp32.
        _reorder("reorder token-major", 10, 3, 5, 3, 777, 80, "f32", 1, True),
        # One sequence, one token, a short context: plain decode, bound by latency.
        _tree("tree single token", 1, 1, 14, 2, 64, 1000, 1000, "bf16", False),
        # Drafted trees of 26 nodes for a small batch with ragged contexts.
        _tree("tree drafted", 8, 26, 15, 5, 64, 4096, 17, "bf16", True),
        # Full trees over long contexts with grouped heads: the largest.
        _tree("tree long context", 4, 64, 32, 8, 128, 32768, 20000, "f16", False),
        # One sequence's accepted tokens, 24 layers of K and V.
        _accept("accept one sequence", 48, 1, 26, 5, 2, 1024, 64, "bf16"),
        # A batch of 64 sequences with full trees.
        _accept("accept batch", 24, 64, 64, 8, 4, 256, 128, "bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["beam", "reorder", "tree", "accept"])
    if op == "beam":
        beams = _log(rng, 1, 32)
        vocab = _log(rng, 500, 160000)
        batch = _log(rng, 1, max(1, min(64, 32 * 8 * 151936 // (beams * vocab))))
        c = _beam("", batch, beams, vocab, rng.randint(1, min(64, 2 * beams)),
                  rng.choice(["f32", "bf16", "f16"]), rng.choice([0, 0, 1, 8, 13]),
                  rng.choice([1.0, 1.0, 0.5, 0.01]))
    elif op == "reorder":
        beams, dim = _log(rng, 2, 32), 8 * rng.randint(1, 16)
        heads, entries = rng.randint(1, 12), _log(rng, 1, 4096)
        row = heads * entries * dim * 4
        batch = _log(rng, 1, max(1, min(32, (1 << 29) // (row * beams))))
        layers = _log(rng, 1, max(1, min(48, (1 << 31) // (row * beams * batch))))
        c = _reorder("", layers, batch, beams, heads, entries, dim,
                     rng.choice(["f32", "bf16", "f16"]), rng.randint(0, entries),
                     rng.random() < 0.5)
    elif op == "tree":
        kv_heads, group = rng.randint(1, 8), rng.randint(1, 8)
        nodes, dim = _log(rng, 1, 64), 8 * rng.randint(2, 16)
        longest = _log(rng, 1, 32768)
        batch = _log(rng, 1, max(1, min(48, 4 * 8 * 32768 // (kv_heads * longest))))
        c = _tree("", batch, nodes, kv_heads * group, kv_heads, dim, longest,
                  rng.randint(0, longest), rng.choice(["bf16", "f16"]), rng.random() < 0.5)
    else:
        nodes, heads = _log(rng, 1, 64), rng.randint(1, 8)
        dim, entries = 8 * rng.randint(1, 16), nodes + _log(rng, 8, 1024)
        row = heads * entries * dim * 4
        batch = _log(rng, 1, max(1, min(64, (1 << 28) // row)))
        layers = _log(rng, 1, max(1, min(48, (1 << 30) // (row * batch))))
        c = _accept("", layers, batch, nodes, rng.randint(1, min(nodes, 8)), heads, entries,
                    dim, rng.choice(["f32", "bf16", "f16"]))
    del c["name"]
    return c


def work(case):
    c, size = case, SIZES[case["dtype"]]
    if c["op"] == "beam":
        n = c["batch"] * c["beams"] * c["vocab"]
        # each logit: a subtraction, an exponential, an addition, a comparison
        return {"bytes": n * size + c["batch"] * (5 * c["beams"] + 17 * c["n_out"]),
                "flops": 4 * n}
    if c["op"] == "reorder":
        k = c["beams"]
        # parents are uniform: a row moves unless it keeps its own place, and a source is
        # read once however many rows take it
        moved = k - 1
        read = k * (1 - (1 - 1 / k) ** (k - 1))
        one = (c["heads"] * c["dim"] * size * (c["entries"] + c["shortest"]) / 2)
        return {"bytes": c["layers"] * c["batch"] * one * (moved + read) + 4, "flops": 0}
    if c["op"] == "tree":
        keys = c["batch"] * ((c["longest"] + c["shortest"]) / 2 + c["nodes"])
        rows = c["batch"] * c["nodes"] * c["heads"] * c["dim"]
        return {"bytes": (2 * keys * c["kv_heads"] * c["dim"] + 2 * rows) * size,
                "flops": 4 * keys * c["nodes"] * c["heads"] * c["dim"]}
    moved = (c["depth"] - 1) / 2  # accepted nodes behind the root, on average
    one = c["heads"] * c["dim"] * size
    return {"bytes": 2 * c["layers"] * c["batch"] * moved * one
            + c["batch"] * (16 * c["nodes"] + 16), "flops": 0}


# -- the inputs --------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed) * 7919 + 13)
    return g


def _lengths(r, batch, shortest, longest):
    n = r.randint(shortest, longest + 1, batch)
    n[0] = longest
    return torch.from_numpy(n.astype(np.int32)).to(DEVICE)


def _random_tree(r, nodes):
    """Parents of a drafted tree: node 0 the root, later nodes below earlier ones, the early
    ones more often; the last slots of some trees unused."""
    p = np.array([-1] + [int(i * r.rand() ** 2) for i in range(1, nodes)], np.int32)
    used = nodes if r.rand() < 0.5 else r.randint(1, nodes + 1)
    p[used:] = -2
    return p


def prepare(case, seed):
    c = dict(case)
    g, r = _generator(seed), np.random.RandomState((int(seed) * 104729 + 7) % (1 << 31))
    s = {"case": c}
    if c["op"] == "beam":
        b, k, v = c["batch"], c["beams"], c["vocab"]
        x = torch.empty(b, k, v + c["pad"], dtype=TYPES[c["dtype"]], device=DEVICE)
        for i in range(b):  # logits of a language model: a wide bell
            x[i] = 4 * torch.randn(k, v + c["pad"], device=DEVICE, generator=g)
            if c["allowed"] < 1:  # what a grammar bans, the same tokens for a prompt's beams
                ban = torch.rand(v + c["pad"], device=DEVICE, generator=g) >= c["allowed"]
                x[i].masked_fill_(ban, -math.inf)
        s["logits"] = x[..., :v]
        scores = -np.sort(r.gamma(4.0, 0.7, (b, k)), axis=1)
        scores -= 6 * r.rand(b, 1)
        first = r.rand(b) < 0.2  # prompts at their first step: one beam lives
        first[0] = False
        scores[first, 1:] = -math.inf
        s["scores"] = torch.from_numpy(scores.astype(np.float32)).to(DEVICE)
        s["finished"] = torch.from_numpy((r.rand(b, k) < 0.15) & ~first[:, None]).to(DEVICE)
        s["eos"] = v - 1
    elif c["op"] == "reorder":
        rows, h, t, d = c["batch"] * c["beams"], c["heads"], c["entries"], c["dim"]
        shape = (c["layers"], rows) + ((t, h, d) if c["token_major"] else (h, t, d))
        x = torch.empty(shape, dtype=TYPES[c["dtype"]], device=DEVICE)
        for layer in x:
            layer.copy_(torch.randn(shape[1:], device=DEVICE, generator=g))
        s["buffer"] = x
        # the layers' states, each as [rows, heads, entries, dim]
        s["states"] = x.transpose(2, 3) if c["token_major"] else x
        p = r.randint(0, c["beams"], (c["batch"], c["beams"]))
        s["parents"] = torch.from_numpy(p.astype(np.int32)).to(DEVICE)
        s["lengths"] = _lengths(r, c["batch"], c["shortest"], t)
    elif c["op"] == "tree":
        b, n, hq, hk, d = c["batch"], c["nodes"], c["heads"], c["kv_heads"], c["dim"]
        t = c["longest"] + n + 5  # the cache holds the longest context, its tree and some more
        dt = TYPES[c["dtype"]]
        s["q"] = torch.randn(b, n, hq, d, device=DEVICE, generator=g).to(dt)
        shape = (b, t, hk, d) if c["token_major"] else (b, hk, t, d)
        for name in ("k", "v"):
            x = torch.empty(shape, dtype=dt, device=DEVICE)
            for i in range(b):
                x[i] = torch.randn(shape[1:], device=DEVICE, generator=g)
            s[name] = x.transpose(1, 2) if c["token_major"] else x
        s["lengths"] = _lengths(r, b, c["shortest"], c["longest"])
        s["parents"] = torch.from_numpy(np.stack([_random_tree(r, n) for _ in range(b)])).to(DEVICE)
    else:
        b, n, t = c["batch"], c["nodes"], c["entries"]
        parents = np.stack([_random_tree(r, n) for _ in range(b)])
        tokens = r.randint(0, 40, (b, n)).astype(np.int32)
        sampled = r.randint(40, 80, (b, n)).astype(np.int32)
        for i in range(b):  # the model agrees with one chain of the tree
            used = int((parents[i] > -2).sum())
            m = r.randint(1, c["depth"] + 1)
            m = min(m, used)
            chain = np.concatenate([[0], 1 + np.sort(r.permutation(used - 1)[:m - 1])]).astype(int)
            parents[i, chain[1:]] = chain[:-1]
            sampled[i, chain[:-1]] = tokens[i, chain[1:]]
        x = torch.empty(c["layers"], b, c["heads"], t, c["dim"], dtype=TYPES[c["dtype"]],
                        device=DEVICE)
        for layer in x:
            layer.copy_(torch.randn(layer.shape, device=DEVICE, generator=g))
        s["buffer"] = x
        s["parents"] = torch.from_numpy(parents).to(DEVICE)
        s["tokens"] = torch.from_numpy(tokens).to(DEVICE)
        s["sampled"] = torch.from_numpy(sampled).to(DEVICE)
        s["lengths"] = _lengths(r, b, 0, t - n)
    return s


# -- the plain forms ---------------------------------------------------------------------
def _plain_beam(s):
    """Scores of all continuations in 64 bits, sorted with the lowest index first on ties."""
    x, scores, done = s["logits"].double(), s["scores"].double(), s["finished"]
    b, k, v = x.shape
    n = s["case"]["n_out"]
    top = x.amax(-1, keepdim=True).clamp_min(-1e300)
    total = top + (x - top).exp().sum(-1, keepdim=True).log()
    key = scores[..., None] + (x - total)
    dead = done | (scores == -math.inf)
    key = torch.where(dead[..., None] | (x == -math.inf), -math.inf, key)
    ids = torch.arange(v, device=x.device)
    key = torch.where((done[..., None]) & (ids == s["eos"]), scores[..., None], key).view(b, k * v)
    best, at = torch.sort(key, dim=-1, descending=True, stable=True)
    missing = n - min(n, k * v)
    best = torch.nn.functional.pad(best[:, :n], (0, missing), value=-math.inf)
    at = torch.nn.functional.pad(at[:, :n], (0, missing))
    none = best == -math.inf
    parent, token = at // v, at % v
    ends = done.gather(1, parent) | (token == s["eos"]) | none
    return {"scores": best.float(), "parents": torch.where(none, -1, parent).int(),
            "tokens": torch.where(none, -1, token).int(), "finished": ends}


def _plain_reorder(s):
    c, x = s["case"], s["buffer"]
    k, t = c["beams"], c["entries"]
    first = torch.arange(c["batch"], device=x.device) * k
    source = (first[:, None] + s["parents"]).reshape(-1)
    kept = torch.arange(t, device=x.device) >= s["lengths"].repeat_interleave(k)[:, None]
    kept = kept[:, :, None, None] if c["token_major"] else kept[:, None, :, None]
    x.copy_(torch.where(kept, x, x[:, source]))
    return x


def _sees(parents):
    """Per node of a tree the slots it sees (itself and its ancestors) and whether it is in
    use: (I + parent matrix)^n counts the paths upwards, a slot in use ends at a -1."""
    n = parents.shape[1]
    i = torch.arange(n, device=parents.device)
    up = ((parents[:, :, None] == i) & (i < i[:, None])).double()
    paths = torch.linalg.matrix_power(torch.eye(n, device=parents.device).double() + up, n)
    sees = paths > 0
    used = (sees & (parents == -1)[:, None, :]).any(-1)
    return sees, used


def _plain_tree(s):
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    b, n, hq, d = q.shape
    hk, t = k.shape[1], k.shape[2]
    pos = torch.arange(t, device=q.device)
    start = s["lengths"].long()[:, None]
    sees, used = _sees(s["parents"])
    used = used & (start + torch.arange(n, device=q.device) < t)
    slot = (pos - start).clamp(0, n - 1)
    tree = sees.gather(2, slot[:, None, :].expand(b, n, t))
    inside = (pos >= start) & (pos < start + n)
    mask = ((pos < start)[:, None, :] | (inside[:, None, :] & tree)) & used[:, :, None]
    v = torch.where((mask.any(1))[:, None, :, None], v, 0)
    q = q.transpose(1, 2).reshape(b, hk, hq // hk * n, d)
    x = (q @ k.transpose(-1, -2)) * d ** -0.5
    x = x.view(b, hq, n, t).masked_fill(~mask[:, None], -math.inf)
    p = (x - x.amax(-1, keepdim=True).clamp_min(-1e30)).exp()
    total = p.sum(-1, keepdim=True)
    o = (p.view(b, hk, hq // hk * n, t) @ v).view(b, hq, n, d)
    o = torch.where(total > 0, o / total, 0)
    return o.transpose(1, 2).contiguous().to(s["q"].dtype)


def _plain_accept(s):
    parents, tokens, sampled = s["parents"].long(), s["tokens"], s["sampled"]
    b, n = parents.shape
    i = torch.arange(n, device=parents.device)
    sees, used = _sees(parents)
    used = used & (s["lengths"].long()[:, None] + i < s["case"]["entries"])
    up = parents.clamp_min(0)
    fits = (parents >= 0) & (sampled.gather(1, up) == tokens) & used
    # of siblings that fit the lowest is taken
    rival = (parents[:, :, None] == parents[:, None, :]) & (i < i[:, None]) & fits[:, None, :]
    taken = (fits & ~rival.any(-1)) | ((i == 0) & (parents == -1) & used)
    accepted = ~(sees & ~taken[:, None, :]).any(-1)
    count = accepted.sum(-1)
    path = torch.where(accepted, i, n).sort(-1).values
    path = torch.where(path < n, path, -1)
    last = path.gather(1, (count - 1).clamp_min(0)[:, None])[:, 0]
    following = torch.where(count > 0, sampled.gather(1, last.clamp_min(0)[:, None])[:, 0], -1)
    x = s["buffer"]
    pos = torch.arange(x.shape[3], device=x.device)
    slot = pos - s["lengths"].long()[:, None]
    moved = (slot >= 0) & (slot < count[:, None])
    source = torch.where(moved, s["lengths"].long()[:, None]
                         + path.gather(1, slot.clamp(0, n - 1)), pos)
    x.copy_(x.gather(3, source[None, :, None, :, None].expand(x.shape)))
    return {"path": path.int(), "counts": count.int(), "next_tokens": following.int(),
            "lengths": (s["lengths"] + count).int(), "caches": x}


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"beam": _plain_beam, "reorder": _plain_reorder, "tree": _plain_tree,
                "accept": _plain_accept}[op](state)
    import tabby_b200

    if op == "beam":
        r = tabby_b200.beam_step(state["logits"], state["scores"], state["case"]["n_out"],
                                 finished=state["finished"], eos_id=state["eos"])
        return {"scores": r.scores, "parents": r.parents, "tokens": r.tokens,
                "finished": r.finished}
    if op == "reorder":
        tabby_b200.reorder_states(state["states"], state["parents"], state["lengths"])
        return state["buffer"]
    if op == "tree":
        return tabby_b200.tree_attention(state["q"], state["k"], state["v"], state["lengths"],
                                         state["parents"])
    r = tabby_b200.tree_accept(state["sampled"], state["tokens"], state["parents"],
                               state["lengths"], state["buffer"])
    return {"path": r.path, "counts": r.counts, "next_tokens": r.next_tokens,
            "lengths": r.lengths, "caches": state["buffer"]}


# -- the definitions in 64 bits -------------------------------------------------------------
def _exact_beam(s):
    """Per prompt: the scores sorted by (score, index) with a two-key sort on the host for the
    candidates that can matter, the best n of each beam."""
    c = s["case"]
    n, v = c["n_out"], c["vocab"]
    scores, done = s["scores"].double().cpu().numpy(), s["finished"].cpu().numpy()
    out = {"scores": np.full((c["batch"], n), -np.inf), "parents": None, "tokens": None,
           "finished": None}
    for b in range(c["batch"]):
        found = []
        for k in range(c["beams"]):
            if scores[b, k] == -np.inf:
                continue
            if done[b, k]:
                found.append((-scores[b, k], k * v + s["eos"]))
                continue
            x = s["logits"][b, k].double()
            if not bool((x > -math.inf).any()):
                continue
            logp = (x - torch.logsumexp(x, 0)).cpu().numpy()
            best = np.argpartition(-logp, min(n, v) - 1)[:n] if n < v else np.arange(v)
            floor = logp[best].min()
            for t in np.nonzero((logp >= floor) & (logp > -np.inf))[0]:
                found.append((-(scores[b, k] + logp[t]), k * v + int(t)))
        for j, (neg, _) in enumerate(sorted(found)[:n]):
            out["scores"][b, j] = -neg
    return out


def _exact_reorder(s):
    c = s["case"]
    x = s["buffer"].double()
    y = x.clone()
    parents, lengths = s["parents"].cpu().tolist(), s["lengths"].cpu().tolist()
    for b in range(c["batch"]):
        for k in range(c["beams"]):
            to, of, m = b * c["beams"] + k, b * c["beams"] + parents[b][k], lengths[b]
            if c["token_major"]:
                y[:, to, :m] = x[:, of, :m]
            else:
                y[:, to, :, :m] = x[:, of, :, :m]
    return y


def _chain(parents, i):
    """Node i and its ancestors, or None where the way up does not end in a root."""
    way = [i]
    while parents[way[-1]] != -1:
        p = parents[way[-1]]
        if p < 0 or p >= way[-1]:
            return None
        way.append(p)
    return way


def _exact_tree(s):
    q, k, v = s["q"], s["k"], s["v"]
    b, n, hq, d = q.shape
    hk, t = k.shape[1], k.shape[2]
    out = torch.zeros(b, n, hq, d, dtype=torch.float64, device=q.device)
    parents, lengths = s["parents"].cpu().tolist(), s["lengths"].cpu().tolist()
    for i in range(b):
        m = min(lengths[i] + n, t)
        ways = [_chain(parents[i], j) if lengths[i] + j < t else None for j in range(n)]
        off = torch.full((n, m), -math.inf, dtype=torch.float64, device=q.device)
        for j, way in enumerate(ways):
            if way is not None:
                off[j, :lengths[i]] = 0
                off[j, [lengths[i] + w for w in way]] = 0
        live = [j for j, way in enumerate(ways) if way is not None]
        seen = torch.zeros(m, 1, dtype=torch.float64, device=q.device)
        seen[(off[live] == 0).any(0)] = 1
        for h in range(hq):
            keys, values = k[i, h * hk // hq, :m].double(), v[i, h * hk // hq, :m].double()
            values = torch.where(seen > 0, values, 0)
            x = q[i, live, h].double() @ keys.T / math.sqrt(d) + off[live]
            out[i, live, h] = torch.softmax(x, -1) @ values
    return out


def _exact_accept(s):
    c = s["case"]
    x = s["buffer"].double()
    parents, lengths = s["parents"].cpu().tolist(), s["lengths"].cpu().tolist()
    tokens, sampled = s["tokens"].cpu().tolist(), s["sampled"].cpu().tolist()
    for b in range(c["batch"]):
        way = [0]
        while True:
            fits = [j for j in range(way[-1] + 1, c["nodes"]) if parents[b][j] == way[-1]
                    and tokens[b][j] == sampled[b][way[-1]] and lengths[b] + j < c["entries"]]
            if not fits:
                break
            way.append(fits[0])
        rows = [lengths[b] + j for j in way]
        x[:, b, :, lengths[b]:lengths[b] + len(way)] = x[:, b, :, rows]
    return {"path": None, "counts": None, "next_tokens": None, "lengths": None, "caches": x}


def exact(case, seed):
    s = prepare(case, seed)
    return {"beam": _exact_beam, "reorder": _exact_reorder, "tree": _exact_tree,
            "accept": _exact_accept}[case["op"]](s)
