"""The operators a server needs between two tokens of an answer: drafted tokens attended as a tree over the cache, verified
against the target model's probabilities, the accepted ones' cache rows moved together; and a cache that accumulates the
attention each key receives and is cut down to its heaviest keys.

Head counts are those of this repository's tests and benchmark: 32 query heads over 8 KV heads, 32 over 32, and 4 over 1 (one
rank of a head-sharded run); cache lengths are its sequence lengths. `own` false: elementary torch operations in 32 bits (64
for sums of probabilities, whose comparisons decide tokens). `own` true: the calls a program makes of the package.
"""
import math
import random

import torch

own = False

D = 128
SCALE = D ** -0.5


class _Layer:
    """The attention module a model hands to the backend: only its layer index is looked at."""
    layer_idx = 0


def _tree(B, n, S, H=32, Hkv=8, tree="chain", fill=1.0, via="call"):
    return {"op": "tree", "B": B, "n": n, "S": S, "H": H, "Hkv": Hkv, "tree": tree, "fill": fill, "via": via}


def _decode(B, S, H=32, Hkv=8, fill=1.0):
    return {"op": "decode", "B": B, "S": S, "H": H, "Hkv": Hkv, "fill": fill}


def _verify(B, n, V, dtype="float32", tree="chain", drafts="sampled"):
    return {"op": "verify", "B": B, "n": n, "V": V, "dtype": dtype, "tree": tree, "drafts": drafts}


def _keep(B, n, S, layers, Hkv=8):
    return {"op": "keep", "B": B, "n": n, "S": S, "layers": layers, "Hkv": Hkv}


def _evict(B, S, keep, recent, Hkv=8, fill=1.0):
    return {"op": "evict", "B": B, "S": S, "keep": keep, "recent": recent, "Hkv": Hkv, "fill": fill}


def listed():
    def named(name, case):
        return dict(case, name=name)

    return [
        # one user's chat: the last token and four drafts of a small model, a chain over a few thousand keys, per layer
        named("tree-chain-one", _tree(1, 5, 3001)),
        # a batch of assisted generations through the backend: static cache, its padding and causality in one boolean mask
        named("tree-backend-16", _tree(16, 8, 4096, fill=0.25, via="backend")),
        # tree of drafts (several guesses at each place) over a batch's caches of different lengths
        named("tree-26-batch-8", _tree(8, 26, 8192, tree="tree", fill=0.5)),
        # the widest tree over a long document
        named("tree-64-long", _tree(1, 64, 65536, tree="tree")),
        # verification for one user: a short chain whose drafts come without probabilities (looked up in the prompt)
        named("verify-chain-one", _verify(1, 9, 50257, "bfloat16", drafts="lookup")),
        # verification of trees for a batch with a large vocabulary
        named("verify-tree-32", _verify(32, 26, 128257, tree="tree")),
        # the accepted rows of one user's cache moved together, 16 layers at once
        named("keep-one", _keep(1, 26, 2048, 16)),
        # and of a batch with the widest trees
        named("keep-batch-8", _keep(8, 64, 1000, 16)),
        # one step of the answer that also accumulates what each key receives
        named("decode-weights-one", _decode(1, 4097)),
        # the same for a batch whose caches are filled to different lengths
        named("decode-weights-16", _decode(16, 8192, fill=0.25)),
        # one user's cache cut to half when it is full
        named("evict-one", _evict(1, 4096, 2048, 512)),
        # a batch's caches, filled to different lengths, cut to a fixed budget
        named("evict-16", _evict(16, 16384, 2048, 256, fill=0.1)),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))

    H, Hkv = rng.choice([(32, 8), (32, 8), (32, 32), (4, 1)])
    op = rng.choice(["tree", "tree", "tree", "verify", "verify", "keep", "decode", "evict"])
    fill = rng.choice([1.0, round(rng.uniform(0.05, 0.95), 3)])
    if op == "tree":
        B = rng.choice([1, 1, 2, 5, 8, 16])
        n = log_int(2, 64)
        S = log_int(n + 1, min(65536 * 8 // (B * Hkv), 65536 * 64 * 32 // (B * n * H)))
        return _tree(B, n, S, H, Hkv, rng.choice(["chain", "tree", "tree"]), fill, rng.choice(["call", "call", "backend"]))
    if op == "decode":
        B = rng.choice([1, 1, 2, 5, 8, 16, 32])
        return _decode(B, log_int(1, 16 * 8192 * 8 // (B * Hkv)), H, Hkv, fill)
    if op == "verify":
        B, n = rng.choice([1, 2, 7, 16, 32]), log_int(2, 40)
        V = log_int(1000, min(152064, 32 * 26 * 128257 // (B * n)))
        return _verify(B, n, V, rng.choice(["float32", "float32", "bfloat16", "float16"]), rng.choice(["chain", "tree"]),
                       rng.choice(["sampled", "sampled", "lookup"]))
    if op == "keep":
        B, n = rng.choice([1, 1, 3, 8]), log_int(2, 64)
        return _keep(B, n, log_int(n + 1, 8192 // B), rng.choice([1, 4, 16]), Hkv)
    B = rng.choice([1, 1, 3, 8, 16])
    S = log_int(2, 16384 * 16 * 8 // (B * Hkv) if B * Hkv > 32 else 65536)
    keep = rng.randint(1, max(1, min(S, 2048 * 16 * 8 // (B * Hkv))))
    return _evict(B, S, keep, rng.randint(0, keep), Hkv, fill)


# ---- inputs -------------------------------------------------------------------------------------------------

def _parents(case, seed):
    """Parent of each node; node 0 is the token sampled last, whose parent is the cache."""
    n = case["n"]
    if case["tree"] == "chain":
        return [i - 1 for i in range(n)]
    rng = random.Random(seed)
    return [-1] + [rng.randint(max(0, i - 9), i - 1) for i in range(1, n)]


def _lengths(g, case, most):
    """Rows in use, between fill * most and most, the first sequence's all."""
    B = case["B"]
    share = case["fill"] + (1 - case["fill"]) * torch.rand(B, generator=g, device="cuda")
    share[0] = 1
    return (most * share).round().int().clamp(0, most)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, dtype=torch.bfloat16):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)

    op, B = case["op"], case["B"]
    state = {"case": case}
    if op in ("tree", "decode"):
        H, Hkv, S = case["H"], case["Hkv"], case["S"]
        n = case.get("n", 1)
        state["q"], state["k"], state["v"] = randn(B, H, n, D), randn(B, Hkv, S, D), randn(B, Hkv, S, D)
        if op == "tree" and case["via"] == "backend":
            # left-padded sequences of different lengths that end at the newest token, drafts included
            import intra_b200.llm_backend
            state["attention"] = intra_b200.llm_backend.make_intra_attention()
            used = _lengths(g, case, S - n) + n
            j = torch.arange(S, device="cuda")
            causal = j[None, :] <= (S - n + torch.arange(n, device="cuda"))[:, None]
            state["mask"] = (causal[None] & (j[None, None, :] >= (S - used)[:, None, None]))[:, None]
            return state
        state["lengths"] = _lengths(g, case, S - n)
        if op == "tree":
            state["parents"] = None if case["tree"] == "chain" else torch.tensor(_parents(case, seed), dtype=torch.int32, device="cuda")
        else:
            # what earlier steps have accumulated
            state["weights"] = torch.rand(B, Hkv, S, generator=g, device="cuda") ** 8 * 4
        return state
    if op == "verify":
        n, V, dtype = case["n"], case["V"], getattr(torch, case["dtype"])
        parents = _parents(case, seed)
        state["parents"] = None if case["tree"] == "chain" else torch.tensor(parents, dtype=torch.int32, device="cuda")
        state["target"] = torch.empty(B, n, V, dtype=dtype, device="cuda")
        state["draft"] = torch.empty(B, n, V, dtype=dtype, device="cuda") if case["drafts"] == "sampled" else None
        state["tokens"] = torch.zeros(B, n, dtype=torch.int64, device="cuda")
        up = torch.tensor(parents, device="cuda").clamp_min(0)
        for b in range(B):
            logits = randn(n, V, dtype=torch.float32) * 3
            state["target"][b] = logits.softmax(-1)
            near = (logits + 0.6 * randn(n, V, dtype=torch.float32)).softmax(-1)      # the small model's opinion
            if state["draft"] is not None:
                state["draft"][b] = near
            guess = torch.multinomial(near[up], 1, generator=g)[:, 0]
            # a looked-up draft repeats the text: mostly the likeliest token
            likely = state["target"][b, up].argmax(-1)
            state["tokens"][b] = guess if state["draft"] is not None else torch.where(torch.rand(n, generator=g, device="cuda") < 0.5, likely, guess)
        state["uniform"] = torch.rand(B, n, generator=g, device="cuda")
        return state
    if op == "keep":
        n, S, Hkv = case["n"], case["S"], case["Hkv"]
        state["caches"] = [randn(B, Hkv, S, D) for _ in range(2 * case["layers"])]
        state["lengths"] = torch.randint(0, S - n + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
        # a path of m nodes after node 0, in increasing order
        chosen = torch.rand(B, n, generator=g, device="cuda") < 0.3
        chosen[:, 0] = True
        place = torch.arange(n, device="cuda").expand(B, n)
        path = torch.where(chosen, place, n).sort(-1).values
        state["path"] = torch.where(path < n, path, -1).int()
        return state
    S, Hkv = case["S"], case["Hkv"]
    state["k"], state["v"] = randn(B, Hkv, S, D), randn(B, Hkv, S, D)
    # few heavy keys, many light ones, some that nothing has ever looked at
    weights = torch.exp(2 * randn(B, Hkv, S, dtype=torch.float32))
    state["weights"] = torch.where(torch.rand(B, Hkv, S, generator=g, device="cuda") < 0.2, 0.0, weights)
    state["lengths"] = _lengths(g, case, S)
    return state


# ---- one pass -----------------------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        return _run_own(state, op)
    if op == "tree":
        visible = state["mask"] if case["via"] == "backend" else _visible(state, case["n"])
        return _attend(state, visible)[0]
    if op == "decode":
        out, p = _attend(state, _visible(state, 1))
        state["weights"] += p.sum((2, 3))
        return out, state["weights"]
    return {"verify": _plain_verify, "keep": _plain_keep, "evict": _plain_evict}[op](state, case)


def _run_own(state, op):
    import intra_b200
    case = state["case"]
    if op == "tree" and case["via"] == "backend":
        return state["attention"](_Layer, state["q"], state["k"], state["v"], state["mask"], scaling=SCALE)[0]
    if op == "tree":
        return intra_b200.tree_attn(state["q"], state["k"], state["v"], state["parents"], state["lengths"])
    if op == "decode":
        out = intra_b200.decode_attn_accumulate(state["q"], state["k"], state["v"], state["weights"], state["lengths"])
        return out, state["weights"]
    if op == "verify":
        return intra_b200.verify_drafts(state["tokens"], state["target"], state["draft"], state["uniform"], state["parents"])
    if op == "keep":
        intra_b200.keep_drafts(state["caches"], state["lengths"], state["path"])
        return state["caches"]
    return intra_b200.evict_cache(state["k"], state["v"], state["weights"], case["keep"], case["recent"], state["lengths"])


def _visible(state, n):
    """(B, 1, n, S): the keys before the n tokens, the ancestors among them, the token itself."""
    S = state["k"].shape[2]
    j = torch.arange(S, device="cuda")
    parents = state.get("parents")
    if parents is None:
        seen = torch.ones(n, n, device="cuda").tril()
    else:
        seen = torch.eye(n, device="cuda")
        seen[1:] += torch.nn.functional.one_hot(parents[1:].long(), n)
        step = 1
        while step < n:                                   # ancestors up to twice as far
            seen = ((seen @ seen) > 0).float()
            step *= 2
    place = j[None, :] - state["lengths"][:, None]        # (B, S): place among the n tokens
    among = (place >= 0) & (place < n)
    own_part = (seen > 0)[:, place.clamp(0, n - 1).long()].transpose(0, 1)
    return ((place < 0)[:, None, :] | (among[:, None, :] & own_part))[:, None]


def _attend(state, visible):
    q, k, v = state["q"], state["k"], state["v"]
    B, H, n, _ = q.shape
    Hkv, S = k.shape[1:3]
    s = torch.matmul(q.float().view(B, Hkv, H // Hkv * n, D), k.float().transpose(-1, -2)).view(B, Hkv, H // Hkv, n, S)
    s = (s * SCALE).masked_fill_(~visible[:, :, None], float("-inf"))
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(B, Hkv, H // Hkv * n, S), v.float()).view(B, H, n, D)
    return out.transpose(1, 2).to(q.dtype).contiguous(), p


def _plain_verify(state, case):
    tokens, target, draft, uniform = state["tokens"], state["target"], state["draft"], state["uniform"].double()
    B, n, V = target.shape
    rows = torch.arange(B, device="cuda")
    if case["tree"] == "chain":
        # drafts up to the first that is rejected
        p = target[:, :-1].gather(2, tokens[:, 1:, None])[..., 0].double()
        q = 1.0 if draft is None else draft[:, :-1].gather(2, tokens[:, 1:, None])[..., 0].double()
        accepted = (uniform[:, 1:] * q < p).long().cumprod(1).sum(1)
        path = torch.arange(n, device="cuda").expand(B, n)
        path = torch.where(path <= accepted[:, None], path, -1)
        left = target[rows, accepted].double()
        after = (accepted + 1).clamp_max(n - 1)
        x = tokens[rows, after][:, None]
        q = torch.zeros_like(left).scatter_(1, x, 1.0) if draft is None else draft[rows, accepted].double()
        rest = (left - q).clamp_min(0)
        rejected = (accepted < n - 1) & (rest.sum(1) > 0)
        left = torch.where(rejected[:, None], rest, left)
    else:
        parents = state["parents"]
        at = torch.zeros(B, dtype=torch.int64, device="cuda")
        accepted = torch.zeros(B, dtype=torch.int64, device="cuda")
        path = torch.full((B, n), -1, dtype=torch.int64, device="cuda")
        path[:, 0] = 0
        left, mass = target[:, 0].double(), torch.ones(B, dtype=torch.float64, device="cuda")
        for i in range(1, n):                             # children stand behind their parents: one pass over the nodes
            child = parents[i] == at
            x = tokens[:, i:i + 1]
            q = torch.zeros_like(left).scatter_(1, x, 1.0) if draft is None else draft[rows, at].double()
            took = child & (uniform[:, i] * q.gather(1, x)[:, 0] * mass < left.gather(1, x)[:, 0])
            rest = (left / mass[:, None] - q).clamp_min(0)
            total = rest.sum(1)
            refused = child & ~took & (total > 0)
            left = torch.where(took[:, None], target[:, i].double(), torch.where(refused[:, None], rest, left))
            mass = torch.where(took, 1.0, torch.where(refused, total, mass))
            accepted = accepted + took
            path[rows, accepted] = torch.where(took, i, path[rows, accepted])
            at = torch.where(took, i, at)
    sums = left.cumsum(1)
    last = torch.searchsorted(sums, uniform[:, :1] * sums[:, -1:], right=True)[:, 0].clamp_max(V - 1)
    out = torch.full_like(tokens, -1)
    out[:, :-1] = torch.where(path >= 0, tokens.gather(1, path.clamp_min(0)), -1)[:, 1:]
    out[rows, accepted] = last
    return accepted.int(), path.int(), out


def _plain_keep(state, case):
    path, B, n = state["path"].long(), case["B"], case["n"]
    to = state["lengths"].long()[:, None] + torch.arange(n, device="cuda")
    source = torch.where(path >= 0, state["lengths"].long()[:, None] + path, to)
    for cache in state["caches"]:
        shape = (B, cache.shape[1], n, D)
        cache.scatter_(2, to[:, None, :, None].expand(shape), cache.gather(2, source[:, None, :, None].expand(shape)))
    return state["caches"]


def _plain_evict(state, case):
    k, v, weights, keep, recent = state["k"], state["v"], state["weights"], case["keep"], case["recent"]
    S = k.shape[2]
    j, used = torch.arange(S, device="cuda"), state["lengths"][:, None, None]
    order = weights.masked_fill(j >= used - recent, float("inf")).masked_fill(j >= used, float("-inf"))
    kept = order.sort(dim=-1, descending=True, stable=True).indices[..., :keep].sort(-1).values
    there = kept < used
    # rows past the length sort behind all others: the kept ones come first
    index = kept[..., None].expand(-1, -1, -1, D)
    k2 = k.gather(2, index).masked_fill(~there[..., None], 0)
    v2 = v.gather(2, index).masked_fill(~there[..., None], 0)
    return k2, v2, weights.gather(2, kept).masked_fill(~there, 0), torch.where(there, kept, -1).int()


# ---- the floor and the truth --------------------------------------------------------------------------------

def work(case):
    op, B = case["op"], case["B"]
    if op in ("tree", "decode"):
        H, Hkv, S, n = case["H"], case["Hkv"], case["S"], case.get("n", 1)
        keys = n + (S - n) * (1 + (B - 1) * (1 + case["fill"]) / 2) / B
        nbytes = 2 * D * B * (2 * H * n + 2 * Hkv * keys)
        nbytes += 8 * B * Hkv * keys if op == "decode" else B * n * S if case["via"] == "backend" else 0
        return {"bytes": nbytes, "flops": 4 * D * B * H * n * keys}
    if op == "verify":
        size = 4 if case["dtype"] == "float32" else 2
        both = 2 if case["drafts"] == "sampled" else 1
        return {"bytes": B * (case["V"] * size * both + case["n"] * (24 + size * both)), "flops": 3 * B * case["V"]}
    if op == "keep":
        moved = 1 + 0.3 * (case["n"] - 1)
        return {"bytes": 2 * case["layers"] * B * case["Hkv"] * moved * 2 * 2 * D, "flops": 0}
    S, Hkv = case["S"], case["Hkv"]
    used = S * (1 + (B - 1) * (1 + case["fill"]) / 2) / B
    return {"bytes": B * Hkv * (4 * used + case["keep"] * (4 * 2 * D + 8)), "flops": 0}


def exact(case, seed):
    op = case["op"]
    if op == "verify":
        return None
    state = prepare(case, seed)
    B = case["B"]
    if op == "keep":
        lengths, path, result = state["lengths"].tolist(), state["path"].tolist(), []
        for cache in state["caches"]:
            moved = cache.double()
            for b in range(B):
                nodes = [i for i in path[b] if i >= 0]
                first = lengths[b]
                moved[b, :, first:first + len(nodes)] = cache[b, :, [first + i for i in nodes]].double()
            result.append(moved)
        return result
    if op == "evict":
        keep, recent, Hkv = case["keep"], case["recent"], case["Hkv"]
        k2, v2 = (torch.zeros(B, Hkv, keep, D, dtype=torch.float64, device="cuda") for _ in range(2))
        w2 = torch.zeros(B, Hkv, keep, dtype=torch.float64, device="cuda")
        for b, used in enumerate(state["lengths"].tolist()):
            for h in range(Hkv):
                w = state["weights"][b, h, :used].double()
                if used > keep:
                    old = used - recent
                    by_weight = w[:old].cpu().numpy()
                    order = sorted(range(old), key=lambda i: (-by_weight[i], i))[:keep - recent]
                    rows = sorted(order) + list(range(old, used))
                else:
                    rows = list(range(used))
                at = torch.tensor(rows, dtype=torch.long, device="cuda")
                k2[b, h, :len(rows)], v2[b, h, :len(rows)] = state["k"][b, h, at].double(), state["v"][b, h, at].double()
                w2[b, h, :len(rows)] = w[at]
        return k2, v2, w2, None
    H, Hkv, S, n = case["H"], case["Hkv"], case["S"], case.get("n", 1)
    rep = H // Hkv
    out = torch.zeros(B, n, H, D, dtype=torch.float64, device="cuda")
    gained = torch.zeros(B, Hkv, S, dtype=torch.float64, device="cuda")
    family = [{i} for i in range(n)]
    if op == "tree":
        for i, up in enumerate(_parents(case if case["via"] == "call" else dict(case, tree="chain"), seed)):
            if up >= 0:
                family[i] |= family[up]
    for b in range(B):
        if case.get("via") == "backend":
            first, before = int((~state["mask"][b, 0, 0]).long().argmin()), S - n
        else:
            first, before = 0, int(state["lengths"][b])
        allowed = torch.zeros(n, before + n - first, dtype=torch.bool, device="cuda")
        allowed[:, :before - first] = True
        for i in range(n):
            allowed[i, [before - first + a for a in family[i]]] = True
        for h in range(Hkv):
            kk, vv = (state[x][b, h, first:before + n].double() for x in "kv")
            s = torch.einsum("rid,jd->rij", state["q"][b, h * rep:(h + 1) * rep].double(), kk) * SCALE
            p = s.masked_fill(~allowed, float("-inf")).softmax(-1)
            out[b, :, h * rep:(h + 1) * rep] = torch.einsum("rij,jd->ird", p, vv)
            gained[b, h, first:before + n] = p.sum((0, 1))
    return out if op == "tree" else (out, state["weights"].double() + gained)
