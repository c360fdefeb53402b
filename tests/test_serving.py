"""The serving operators against plain implementations in 64 bits: attention of drafted tokens, their verification, moving the
accepted rows, the decode step that accumulates weights, eviction; what they refuse; and a step of all of them together."""
import json
import os
import random
import subprocess
import sys

import pytest
import torch

import intra_b200
from intra_b200 import decode_attn_accumulate, evict_cache, keep_drafts, tree_attn, verify_drafts
from intra_b200.llm_backend import make_intra_attention

SCALE = 128 ** -0.5
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _cache(B, Hkv, S, seed, layout="bhsd", device="cuda"):
    g = _gen(seed)
    shape = {"bhsd": (B, Hkv, S, 128), "bshd": (B, S, Hkv, 128), "sliced": (B, Hkv, S + 40, 128), "batch1": (1, Hkv, S, 128)}[layout]
    k, v = (torch.randn(*shape, generator=g).to(torch.bfloat16).to(device) for _ in range(2))
    if layout == "bshd":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    if layout == "sliced":                                   # a cache that is longer than what is filled
        k[:, :, :3], v[:, :, :3], k[:, :, S + 3:], v[:, :, S + 3:] = (float("nan"),) * 4
        k, v = k[:, :, 3:S + 3], v[:, :, 3:S + 3]
    if layout == "batch1":
        k, v = k.expand(B, -1, -1, -1), v.expand(B, -1, -1, -1)
    return k, v


def _queries(B, H, n, seed, layout="bhnd", device="cuda"):
    x = torch.randn(B, n, H, 128, generator=_gen(seed + 1000)).to(torch.bfloat16).to(device).transpose(1, 2)
    return x.contiguous() if layout == "bhnd" else x


def _parents(kind, B, n, seed):
    """Lists of parents per sequence, or None for a chain given as such."""
    rng = random.Random(seed)
    if kind is None:
        return None
    if kind == "chain":
        return [[i - 1 for i in range(n)]] * B
    if kind == "star":
        return [[-1] + [0] * (n - 1)] * B
    if kind == "forest":                                     # several roots, and parents that are none: itself, later ones
        return [[rng.choice([-1, -7, i, i + 1, rng.randint(-1, max(i - 1, -1))]) for i in range(n)] for _ in range(B)]
    return [[-1] + [rng.randint(max(0, i - 5), i - 1) for i in range(1, n)] for _ in range(B)]


def _ancestors(parents, n):
    family = []
    for i in range(n):
        up = parents[i] if parents is not None else i - 1
        family.append(({i} | family[up]) if 0 <= up < i else {i})
    return family


def _visible(B, n, S, parents, lengths, mask):
    """(B, n, S) from the definition."""
    seen = torch.zeros(B, n, S, dtype=torch.bool)
    for b in range(B):
        ctx = S - n if lengths is None else min(max(lengths[b], 0), S - n)
        family = _ancestors(None if parents is None else parents[b], n)
        for i in range(n):
            seen[b, i, :ctx] = True
            seen[b, i, [ctx + a for a in family[i]]] = True
    if mask is not None:
        seen &= mask[:, 0, :, :S].cpu()
    return seen.cuda()


def _reference(q, k, v, visible):
    """fp64 result and sum_j p_j |v_j|, both (B, n, H, 128), and the probabilities; hidden keys take no part, whatever they hold."""
    rep = q.shape[1] // k.shape[1]
    gone = ~visible.any(1)[:, None, :, None]
    k, v = k.double().masked_fill(gone, 0).repeat_interleave(rep, 1), v.double().masked_fill(gone, 0).repeat_interleave(rep, 1)
    s = (q.double() @ k.transpose(-1, -2)) * SCALE
    s = s.masked_fill(~visible[:, None], float("-inf"))
    p = torch.where(visible.any(-1)[:, None, :, None], s, 0.0).softmax(-1).masked_fill(~visible[:, None], 0)
    return (p @ v).transpose(1, 2), (p @ v.abs()).transpose(1, 2), p


# Half a bf16 step of the result (2^-9 |ref|) and probabilities kept to 16 bits (each off by 2^-17, their sum by 2^-24 a term; the
# exponential's argument, fp32 products of up to a few hundred, by 2^-16): a factor two on the first, 2^-14 for the rest. Where
# more than 128 rows share a KV head probabilities are bf16 (2^-9 each) and so is a bound on what that makes of the sum; two again.
def _check(out, ref, spread, rows):
    assert bool(out.isfinite().all())
    excess = (out.double() - ref).abs() - (2.0 ** -8 * ref.abs() + (2.0 ** -14 if rows <= 128 else 2.0 ** -8) * spread)
    assert float(excess.max()) <= 0


TREES = [
    # B, H, Hkv, n, S, cache layout, parents, lengths, mask
    (1, 32, 8, 1, 1, "bhsd", None, False, None), (1, 32, 8, 2, 2, "bhsd", None, False, None),
    (1, 32, 8, 4, 300, "bhsd", None, False, None), (1, 32, 8, 5, 3001, "bshd", "chain", True, None),
    (2, 8, 2, 4, 64, "sliced", "random", True, None), (3, 8, 8, 16, 65, "bhsd", "random", True, "padding"),
    (2, 32, 8, 8, 1000, "bhsd", "random", True, "random"), (2, 8, 8, 33, 200, "bshd", "star", True, None),
    (1, 32, 8, 64, 64, "bhsd", "random", False, None), (2, 32, 8, 64, 777, "bhsd", "forest", True, None),
    (1, 32, 8, 64, 5000, "bhsd", "random", True, "random"), (4, 4, 1, 26, 2049, "batch1", "random", True, "shared"),
    (2, 9, 1, 7, 500, "bhsd", "random", True, "strided"), (1, 64, 2, 3, 130, "bhsd", "random", True, "padding"),
    (1, 4, 1, 9, 40000, "sliced", "random", False, None), (16, 32, 8, 8, 2100, "bhsd", None, False, "padding"),
    (70, 4, 1, 3, 90, "bhsd", "random", True, None), (1, 40, 1, 64, 333, "bhsd", "random", True, "random"),
    (2, 32, 8, 20, 16400, "bhsd", "random", True, "padding"),
    # more than 256 rows per KV head, of which the last tile has none; CTAs that hold many whole units, or parts of two
    (1, 5, 1, 64, 900, "bhsd", "random", True, None), (2, 12, 4, 60, 1500, "bshd", "random", True, None), (50, 8, 2, 20, 420, "bhsd", "random", True, None),
    (60, 8, 1, 40, 140, "bhsd", "random", True, None), (130, 8, 2, 33, 400, "sliced", "chain", True, None),
    # caches that tensor maps do not describe
    (3, 8, 2, 30, 1000, "batch1", "random", True, None), (3, 8, 2, 64, 1300, "batch1", None, False, None)]


def _tree_case(B, H, Hkv, n, S, layout, kind, with_lengths, mask_kind, seed=0):
    k, v = _cache(B, Hkv, S, seed, layout)
    q = _queries(B, H, n, seed, "bnhd" if seed % 2 else "bhnd")
    parents = _parents(kind, B, n, seed)
    rng = random.Random(seed)
    lengths = [rng.randint(0, S - n) for _ in range(B)] if with_lengths else None
    if lengths:
        lengths[0] = S - n
        if B > 1:
            lengths[1] = 0
    mask = None
    g = _gen(seed + 5)
    if mask_kind == "padding":
        mask = (torch.arange(S)[None] >= (S * 0.6 * torch.rand(B, 1, generator=g)).long())[:, None, None]
    elif mask_kind == "shared":
        mask = (torch.rand(1, n, S + 3, generator=g) < 0.5)[:, None]
    elif mask_kind == "strided":
        mask = (torch.rand(B, n, 2 * S, generator=g) < 0.5)[:, None, :, ::2]
    elif mask_kind == "random":
        mask = (torch.rand(B, n, S, generator=g) < 0.4)[:, None]
    if mask is not None:
        mask = mask.cuda() if mask_kind != "strided" else mask.contiguous().repeat_interleave(2, -1).cuda()[..., ::2]
    as_int = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda")
    return q, k, v, parents, lengths, mask, as_int(parents), as_int(lengths)


@pytest.mark.gpu
@pytest.mark.parametrize("case", TREES, ids=lambda c: "-".join(map(str, c)))
def test_tree_attention_vs_fp64(case):
    B, H, Hkv, n, S = case[:5]
    q, k, v, parents, lengths, mask, up, used = _tree_case(*case, seed=TREES.index(case))
    out = tree_attn(q, k, v, up, used, mask)
    assert out.shape == (B, n, H, 128) and out.is_contiguous()
    visible = _visible(B, n, S, parents, lengths, mask)
    ref, spread, _ = _reference(q, k, v, visible)
    _check(out, ref, spread, n * H // Hkv)
    assert not bool(out[~visible.any(-1)].any()), "a token that sees nothing gets zeros"
    assert torch.equal(out, tree_attn(q, k, v, up, used, mask)), "two runs differ"
    if up is not None and all(p == parents[0] for p in parents):
        assert torch.equal(out, tree_attn(q, k, v, up[0].contiguous(), used, mask))


@pytest.mark.gpu
@pytest.mark.parametrize("n,rep", [(3, 4), (8, 4), (30, 4), (64, 4)])
def test_what_tokens_do_not_see_does_not_reach_them(n, rep):
    B, Hkv, S = 2, 2, 300
    k, v = _cache(B, Hkv, S, 3)
    q = _queries(B, rep * Hkv, n, 3)
    used = torch.tensor([200, 117], dtype=torch.int32, device="cuda")
    up = torch.tensor([-1] + [0] * (n - 1), dtype=torch.int32, device="cuda")
    want = tree_attn(q, k, v, up, used)
    k2, v2 = k.clone(), v.clone()
    for b, first in enumerate(used.tolist()):                # rows behind the tokens' own hold anything
        k2[b, :, first + n:], v2[b, :, first + n:] = float("nan"), float("inf")
    assert torch.equal(tree_attn(q, k2, v2, up, used), want)
    mask = torch.ones(B, 1, n, S, dtype=torch.bool, device="cuda")
    mask[:, :, :, 50] = False                                # a key hidden from all
    hidden = tree_attn(q, k, v, up, used, mask)
    k2[:, :, 50], v2[:, :, 50] = float("nan"), float("nan")
    assert torch.equal(tree_attn(q, k2, v2, up, used, mask), hidden)
    # a sibling's key holds anything: only that token sees it
    k3, v3 = k.clone(), v.clone()
    k3[0, :, 200 + n - 1], v3[0, :, 200 + n - 1] = float("inf"), float("nan")
    v3[1, :, 117 + n - 1] = float("-inf")
    out = tree_attn(q, k3, v3, up, used)
    assert bool(out[0, -1].isnan().all()) and bool((out[1, -1] == float("-inf")).all())
    ref, spread, _ = _reference(q, k, v, _visible(B, n, S, [up.tolist()] * B, used.tolist(), None))
    _check(out[:, :-1], ref[:, :-1], spread[:, :-1], n * rep)
    # lengths outside the cache are brought into range
    far = torch.tensor([S + 1000, -5], dtype=torch.int32, device="cuda")
    near = torch.tensor([S - n, 0], dtype=torch.int32, device="cuda")
    assert torch.equal(tree_attn(q, k, v, up, far), tree_attn(q, k, v, up, near))


@pytest.mark.gpu
def test_tree_attention_in_a_long_cache():
    """Row offsets past 2^31 elements: a view of a wide buffer, of which few pages are touched."""
    S, n = 40, 5
    wide = torch.empty(S, 1 << 26, dtype=torch.bfloat16, device="cuda")          # 5.4 GB, rows 2^26 elements apart
    k, v = _cache(1, 1, S, 9)
    wide[:, :128], wide[:, 1024:1152] = k[0, 0], v[0, 0]
    kw, vw = wide[:, :128][None, None], wide[:, 1024:1152][None, None]
    q = _queries(1, 4, n, 9)
    assert torch.equal(tree_attn(q, kw, vw), tree_attn(q, k, v))
    weights, want = torch.zeros(2, 1, 1, S, device="cuda")
    assert torch.equal(decode_attn_accumulate(q[:, :, :1], kw, vw, weights), decode_attn_accumulate(q[:, :, :1], k, v, want))
    assert torch.equal(weights, want)
    got = evict_cache(kw, vw, want, 17, 3)
    for a, b in zip(got, evict_cache(k, v, want, 17, 3)):
        assert torch.equal(a, b)
    keep_drafts([kw, vw], torch.tensor([30], dtype=torch.int32, device="cuda"), torch.tensor([[0, 3, 4, -1]], dtype=torch.int32, device="cuda"))
    assert torch.equal(kw[0, 0, 31:32], k[0, 0, 33:34]) and torch.equal(kw[0, 0, 33], k[0, 0, 33])


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hkv,n,S,kind", [(32, 8, 8, 700, "padding"), (8, 8, 5, 129, "random"), (32, 8, 64, 400, "padding"),
                                            (32, 8, 6, 640, None), (8, 2, 4, 300, "bidirectional")])
def test_backend_takes_a_few_tokens_behind_a_cache(H, Hkv, n, S, kind):
    B = 3
    q, (k, v), fn = _queries(B, H, n, 4), _cache(B, Hkv, S, 4), make_intra_attention()
    j, i = torch.arange(S), torch.arange(n)
    seen = (j[None] <= (S - n + i)[:, None]).expand(B, n, S).clone()
    if kind == "padding":
        seen &= (j[None] >= torch.tensor([0, 100, 37])[:, None])[:, None]
    elif kind == "random":                                   # a row that sees nothing among them
        seen &= torch.rand(B, n, S, generator=_gen(1)) < 0.5
        seen[1, 2] = False
    elif kind == "bidirectional":                            # the mask decides alone
        seen[:] = True
    mask = None if kind is None else seen[:, None].cuda()
    out, w = fn(None, q, k, v, mask, scaling=SCALE)
    assert w is None
    ref, spread, _ = _reference(q, k, v, seen.cuda())
    _check(out, ref, spread, n * H // Hkv)
    with torch.enable_grad():
        again, _ = fn(None, q.clone().requires_grad_(True), k, v, mask, scaling=SCALE)
    assert torch.equal(again, out) and not again.requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 4, 20])
def test_backend_takes_masks_the_kernel_does_not(n):
    """Additive masks and masks per head, one token or a few behind a cache."""
    B, H, Hkv, S = 2, 8, 2, 150
    q, (k, v), fn = _queries(B, H, n, 6), _cache(B, Hkv, S, 6), make_intra_attention()
    seen = (torch.rand(B, H, n, S + 4, generator=_gen(n)) < 0.6).cuda()
    seen[..., 0] = True
    for given in (seen, seen[:, :1]):
        additive = torch.zeros(given.shape, dtype=torch.bfloat16, device="cuda").masked_fill(~given, torch.finfo(torch.bfloat16).min)
        s = q.double() @ k.double().repeat_interleave(H // Hkv, 1).transpose(-1, -2) * SCALE
        p = s.masked_fill(~given[..., :S], float("-inf")).softmax(-1)
        vv = v.double().repeat_interleave(H // Hkv, 1)
        ref, spread = (p @ vv).transpose(1, 2), (p @ vv.abs()).transpose(1, 2)
        for mask in (additive, given):
            out, w = fn(None, q, k, v, mask, scaling=SCALE)
            assert w is None and out.shape == (B, n, H, 128)
            # SDPA's probabilities are bf16 numbers (half a step each, 2^-9), and so may its scores be (up to 8: 2^-6 absolute)
            excess = (out.double() - ref).abs() - (2.0 ** -8 * ref.abs() + 2.0 ** -5 * spread)
            assert float(excess.max()) <= 0


def _recipe():
    """Runs what the backend's documentation says a user runs before the model is made."""
    from intra_b200 import llm_backend
    lines = [x.strip() for x in llm_backend.__doc__.splitlines() if x.startswith("    ")]
    assert lines[-1].startswith("model =")
    exec("\n".join(lines[:-1]), {"make_intra_attention": make_intra_attention})


def _small_model(name, device, dtype):
    from transformers import LlamaConfig, LlamaForCausalLM
    config = LlamaConfig(hidden_size=64, num_attention_heads=8, num_key_value_heads=2, head_dim=128, num_hidden_layers=2, intermediate_size=64,
                         vocab_size=50, attn_implementation=name)
    torch.manual_seed(0)
    return config, LlamaForCausalLM(config).to(device, dtype).eval()


def _few_tokens_at_a_time(config, model, cache_kind, padded, chunks=(20, 5, 1, 12)):
    """A left-padded batch and its cache through the model, some tokens at a time. Yields (tokens before, tokens, padding) of each call."""
    from transformers import DynamicCache, StaticCache
    cache = StaticCache(config=config, max_cache_len=96) if cache_kind == "static" else DynamicCache(config=config)
    pad, before, device = [7, 0, 3] if padded else [0, 0, 0], 0, model.device
    for n in chunks:
        mask = (torch.arange(before + n)[None] >= torch.tensor(pad)[:, None]).long().to(device)
        with torch.no_grad():
            model(torch.randint(50, (3, n), generator=_gen(n)).to(device), attention_mask=mask, past_key_values=cache, use_cache=True)
        yield before, n, pad
        before += n


def test_backend_asks_for_masks():
    """The documented registration gives every call of a few tokens a mask, with any cache; a name without one is refused, and
    does not get the unfilled rows of a static cache for keys."""
    pytest.importorskip("transformers")
    from transformers import AttentionInterface
    _recipe()
    fn, seen = make_intra_attention(), []

    def record(module, query, key, value, attention_mask=None, scaling=None, **kw):
        seen.append(None if attention_mask is None else (attention_mask.dtype, tuple(attention_mask.shape)))
        return torch.zeros(query.shape[0], query.shape[2], query.shape[1], 128), None

    AttentionInterface.register("intra_b200", record)
    try:
        for kind in ("static", "dynamic"):
            config, model = _small_model("intra_b200", "cpu", torch.float32)
            for before, n, _ in _few_tokens_at_a_time(config, model, kind, False):
                if before and n > 1:
                    S = 96 if kind == "static" else before + n
                    assert seen == [(torch.bool, (3, 1, n, S))] * 2
                seen.clear()
    finally:
        AttentionInterface.register("intra_b200", fn)
    AttentionInterface.register("intra_b200_without_masks", fn)
    config, model = _small_model("intra_b200_without_masks", "cpu", torch.float32)
    with pytest.raises(ValueError, match="sdpa_mask"):
        next(_few_tokens_at_a_time(config, model, "static", False))


@pytest.mark.gpu
@pytest.mark.parametrize("padded", [False, True])
@pytest.mark.parametrize("kind", ["static", "dynamic"])
def test_a_model_through_the_documented_registration(kind, padded):
    """Every call of a model's attention with a few tokens, or one, behind a cache sees what has been filled and is no padding."""
    pytest.importorskip("transformers")
    from transformers import AttentionInterface
    _recipe()
    fn, calls = make_intra_attention(), []

    def record(module, query, key, value, attention_mask=None, **kw):
        out = fn(module, query, key, value, attention_mask, **kw)
        calls.append((query.clone(), key.clone(), value.clone(), out[0].clone()))
        return out

    AttentionInterface.register("intra_b200", record)
    try:
        config, model = _small_model("intra_b200", "cuda", torch.bfloat16)
        for before, n, pad in _few_tokens_at_a_time(config, model, kind, padded):
            if before or kind == "static":                   # else a prompt, which the patterns take
                assert len(calls) == 2
                for q, k, v, out in calls:
                    j, i = torch.arange(k.shape[2]), torch.arange(n)
                    visible = ((j[None] <= (before + i)[:, None])[None] & (j[None] >= torch.tensor(pad)[:, None])[:, None]).cuda()
                    ref, spread, _ = _reference(q, k, v, visible)
                    real = (before + i[None] >= torch.tensor(pad)[:, None]).cuda()
                    _check(out[real], ref[real], spread[real], 4 * n)
            calls.clear()
    finally:
        AttentionInterface.register("intra_b200", fn)


def _verify_reference(tokens, target, draft, uniform, parents):
    """The definition in Python floats (64 bits), one sequence at a time."""
    accepted, paths, outs = [], [], []
    B, n, V = target.shape
    target = target.double().cpu()
    draft = None if draft is None else draft.double().cpu()
    tokens, uniform = tokens.cpu().tolist(), uniform.double().cpu().tolist()
    for b in range(B):
        up = parents[b] if parents is not None else [i - 1 for i in range(n)]
        at, path, left, Z = 0, [0], target[b, 0], 1.0
        for i in range(1, n):
            if up[i] != at:
                continue
            x = tokens[b][i]
            inside = 0 <= x < V
            if draft is not None:
                q = draft[b, at]
            else:
                q = torch.zeros(V, dtype=torch.float64)
                if inside:
                    q[x] = 1
            qx = float(q[x]) if inside else (1.0 if draft is None else 0.0)
            if uniform[b][i] * qx * Z < (float(left[x]) if inside else 0.0):
                at, left, Z = i, target[b, i], 1.0
                path.append(i)
            else:
                rest = (left / Z - q).clamp_min(0)
                if float(rest.sum()) > 0:
                    left, Z = rest, float(rest.sum())
        sums = left.cumsum(0)
        drawn = int(torch.searchsorted(sums, uniform[b][0] * float(sums[-1]), right=True).clamp_max(V - 1))
        accepted.append(len(path) - 1)
        outs.append([tokens[b][i] for i in path[1:]] + [drawn] + [-1] * (n - len(path)))
        paths.append(path + [-1] * (n - len(path)))
    return torch.tensor(accepted, dtype=torch.int32), torch.tensor(paths, dtype=torch.int32), torch.tensor(outs)


def _verify_case(B, n, V, dtype, kind, drafts, seed, near=0.6):
    g = _gen(seed)
    logits = torch.randn(B, n, V, generator=g) * 2
    target = logits.softmax(-1).to(dtype)
    draft = (logits + near * torch.randn(B, n, V, generator=g)).softmax(-1).to(dtype) if drafts != "lookup" else None
    parents = _parents(kind, B, n, seed)
    tokens = torch.randint(V, (B, n), generator=g)
    for b in range(B):
        for i in range(1, n):
            up = parents[b][i] if parents is not None else i - 1
            if 0 <= up < i:
                row = draft[b, up].float() if draft is not None else target[b, up].float()
                tokens[b, i] = int(torch.multinomial(row, 1, generator=g))
    if draft is not None and drafts == "short":
        draft = draft[:, :-1]
    return tokens, target, draft, torch.rand(B, n, generator=g), parents


@pytest.mark.gpu
@pytest.mark.parametrize("B,n,V,dtype,kind,drafts", [
    (1, 1, 1, torch.float32, None, "sampled"), (1, 1, 100, torch.float32, None, "lookup"), (3, 2, 7, torch.float32, None, "short"),
    (5, 6, 1000, torch.float32, None, "short"), (40, 9, 257, torch.bfloat16, None, "lookup"), (40, 9, 511, torch.float16, None, "short"),
    (64, 26, 333, torch.float32, "random", "sampled"), (64, 26, 2049, torch.bfloat16, "random", "short"), (64, 12, 600, torch.float32, "star", "sampled"),
    (64, 12, 50, torch.float16, "star", "lookup"), (30, 64, 129, torch.float32, "random", "lookup"), (30, 20, 200, torch.float32, "forest", "sampled"),
    (4, 5, 70001, torch.float32, "random", "sampled"), (200, 4, 3000, torch.float32, "star", "sampled")])
def test_verification_vs_the_definition(B, n, V, dtype, kind, drafts):
    tokens, target, draft, uniform, parents = _verify_case(B, n, V, dtype, kind, drafts, B + n + V)
    want = _verify_reference(tokens, target, draft, uniform, parents)
    up = None if parents is None else torch.tensor(parents, dtype=torch.int32).cuda()
    got = verify_drafts(tokens.cuda(), target.cuda(), None if draft is None else draft.cuda(), uniform.cuda(), up)
    for a, b in zip(got, want):
        assert a.dtype == b.dtype and torch.equal(a.cpu(), b)
    # strided inputs, 32-bit tokens: the same
    wide = torch.zeros(B, n + 2, V + 3, dtype=dtype, device="cuda")
    wide[:, 1:-1, 1:-2] = target.cuda()
    again = verify_drafts(tokens.int().cuda(), wide[:, 1:-1, 1:-2], None if draft is None else draft.cuda(), uniform.cuda(), up)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.gpu
def test_verification_at_its_edges():
    V = 1000
    tokens, target, draft, uniform, _ = (x if x is None else x.cuda() for x in _verify_case(4, 5, V, torch.float32, None, "sampled", 1))
    # the drafts' distribution equal to the target's: everything is accepted, whatever the numbers below one
    accepted, path, out = verify_drafts(tokens, target, target, uniform * 0 + 1 - 2 ** -24)
    assert accepted.tolist() == [4] * 4 and torch.equal(path, torch.arange(5, device="cuda", dtype=torch.int32).expand(4, 5))
    assert torch.equal(out[:, :4], tokens[:, 1:])
    # a draft that the target excludes is rejected even by the number zero; nothing of it is drawn
    target2 = target.clone()
    target2[:, 0].scatter_(1, tokens[:, 1:2], 0.0)
    for u in (0.0, 0.5, 1 - 2 ** -24):
        accepted, path, out = verify_drafts(tokens, target2, draft, torch.full_like(uniform, u))
        assert accepted.tolist() == [0] * 4 and bool((out[:, 0] != tokens[:, 1]).all()) and bool((out[:, 1:] == -1).all())
        assert bool((target2[torch.arange(4), 0, out[:, 0]] > 0).all())
    # nothing left (the draft takes more of every token than the target gives): the target's own distribution stands
    short = target * 0.5
    short[:, 0].scatter_(1, tokens[:, 1:2], 0.0)
    got = verify_drafts(tokens, short, target, uniform)
    want = _verify_reference(tokens, short, target, uniform, None)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want)) and got[0].tolist() == [0] * 4
    # zeros of either sign
    sparse = torch.where(torch.rand(target.shape, generator=_gen(2)).cuda() < 0.9, -0.0, target)
    got = verify_drafts(tokens, sparse, draft, uniform)
    want = _verify_reference(tokens, sparse, draft, uniform, None)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want))
    # drafts outside the vocabulary are rejected, and nothing outside the rows is read
    bad = tokens.clone()
    bad[0, 1], bad[1, 1], bad[2, 2] = -1, V, 2 ** 40
    got = verify_drafts(bad, target, None, uniform)
    want = _verify_reference(bad, target, None, uniform, None)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want))
    # a row without any mass, and one of NaN: a token of the vocabulary all the same
    for row in (torch.zeros_like(target), torch.full_like(target, float("nan"))):
        accepted, path, out = verify_drafts(tokens, row, draft, uniform)
        assert accepted.tolist() == [0] * 4 and bool(((out[:, 0] >= 0) & (out[:, 0] < V)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,V", [(1, 1000), (1, 5000), (1, 70001), (200, 3000)])
@pytest.mark.parametrize("drafts", ["none", "lookup", "sampled"])
def test_last_token_of_sparse_rows(dtype, B, V, drafts):
    """Targets of which all but a few tokens at the end are zero, and numbers down to zero: what is drawn has a probability."""
    n = 1 if drafts == "none" else 2
    target, uniform = torch.zeros(B, n, V, dtype=dtype), torch.zeros(B, n)
    for b in range(B):
        target[b, :, V - 4 - (7 * b) % 60] = 0.25
        target[b, :, V - 2] = 0.75
    draft = None
    tokens = torch.full((B, n), 11)                          # which the target excludes
    if drafts == "sampled":
        draft = torch.full((B, n, V), 2.0 ** -13, dtype=dtype)
        draft[:, :, 11] = 0.5
    for u in (0.0, 2.0 ** -149, 2.0 ** -100, 0.2, 0.5, 1 - 2.0 ** -24):
        uniform[:, 0] = u
        want = _verify_reference(tokens, target, draft, uniform, None)
        got = verify_drafts(tokens.cuda(), target.cuda(), None if draft is None else draft.cuda(), uniform.cuda())
        assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want)), u


@pytest.mark.gpu
def test_verification_down_to_the_smallest_probabilities():
    """fp32 denormals count: in a row's sum, and as all that a rejection leaves."""
    V = 1000
    target, uniform, tokens = torch.zeros(1, 2, V), torch.zeros(1, 2), torch.tensor([[0, 640]])
    target[0, :, 300], target[0, :, 640], target[0, :, 900] = 1e-42, 0.5, 0.5
    for u in (0.0, 2.0 ** -149, 0.3):
        uniform[0, 0] = u
        want = _verify_reference(tokens[:, :1], target[:, :1], None, uniform[:, :1], None)
        got = verify_drafts(tokens[:, :1].cuda(), target[:, :1].cuda(), None, uniform[:, :1].cuda())
        assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want)), u
    draft = target * 2                                       # takes more of every token than there is, but for one
    draft[:, :, 300] = 0
    uniform[0, 1] = 1 - 2.0 ** -24
    want = _verify_reference(tokens, target, draft, uniform, None)
    got = verify_drafts(tokens.cuda(), target.cuda(), draft.cuda(), uniform.cuda())
    assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want)) and want[2].tolist() == [[300, -1]]


@pytest.mark.gpu
def test_an_empty_remainder_of_a_long_row():
    """Nothing is left of a row of 2^28 tokens: their zeros do not add up to something, and the row itself stands."""
    V = 1 << 28
    row = torch.zeros(V, device="cuda")
    row[V - 5] = 0.25                                        # a row that sums to a quarter
    tokens, uniform = torch.tensor([[0, V - 5]], device="cuda"), torch.tensor([[0.5, 0.5]], device="cuda")
    accepted, path, out = verify_drafts(tokens, row.expand(1, 2, V), None, uniform)
    assert accepted.tolist() == [0] and path.tolist() == [[0, -1]] and out.tolist() == [[V - 5, -1]]


@pytest.mark.gpu
def test_verified_tokens_are_distributed_as_the_target():
    """First tokens over many draws of drafts and numbers against the target's probabilities: five standard deviations."""
    N, V, n = 40000, 12, 4
    g = torch.Generator(device="cuda").manual_seed(3)
    target = torch.randn(1, n, V, generator=g, device="cuda").mul(1.5).softmax(-1).expand(N, n, V)
    draft = torch.randn(1, n, V, generator=g, device="cuda").mul(1.5).softmax(-1).expand(N, n, V)
    up = torch.tensor([-1, 0, 0, 1], dtype=torch.int32, device="cuda")
    tokens = torch.stack([torch.multinomial(draft[0, max(p, 0)], N, True, generator=g) for p in up.tolist()], 1)
    _, _, out = verify_drafts(tokens, target, draft, torch.rand(N, n, generator=g, device="cuda"), up)
    p = target[0, 0].double()
    seen = torch.bincount(out[:, 0], minlength=V).double() / N
    assert bool(((seen - p).abs() <= 5 * (p * (1 - p) / N).sqrt()).all())


@pytest.mark.gpu
@pytest.mark.parametrize("B,Hkv,S,n,layers,layout", [(1, 1, 1, 1, 1, "bhsd"), (3, 2, 70, 9, 3, "bhsd"), (2, 8, 200, 64, 33, "bshd"),
                                                     (5, 1, 64, 64, 2, "sliced")])
def test_accepted_rows_move_together(B, Hkv, S, n, layers, layout):
    rng = random.Random(n)
    caches = [x for i in range(layers) for x in _cache(B, Hkv, S, i, layout)]
    lengths = [rng.randint(0, S - n) for _ in range(B)]
    paths = []
    for b in range(B):
        nodes = [0] + sorted(rng.sample(range(1, n), rng.randint(0, n - 1)))
        paths.append(nodes + [-1] * (n - len(nodes)))
    if B > 2:
        rng.shuffle(paths[2])                                # any order, gaps
        paths[0][-1], lengths[1] = n + 5, S - n + 1          # no such node; no such rows
    want = []
    for x in caches:
        y = x.clone()
        for b in range(B):
            for i, node in enumerate(paths[b]):
                if 0 <= node < n and lengths[b] <= S - n:
                    y[b, :, lengths[b] + i] = x[b, :, lengths[b] + node]
        want.append(y)
    if layers == 3:                                          # layouts of two kinds in one call
        caches[1] = caches[1].transpose(1, 2).contiguous().transpose(1, 2)
    keep_drafts(caches, torch.tensor(lengths, dtype=torch.int32).cuda(), torch.tensor(paths, dtype=torch.int32).cuda())
    for x, y in zip(caches, want):
        assert torch.equal(x, y)


@pytest.mark.gpu
@pytest.mark.parametrize("B,H,Hkv,S,layout,with_lengths,mask", [
    (1, 32, 8, 1, "bhsd", False, None), (1, 32, 8, 17, "bshd", True, None), (2, 8, 8, 300, "sliced", True, "random"),
    (1, 32, 8, 4097, "bhsd", False, None), (3, 36, 2, 500, "bhsd", True, "padding"), (1, 4, 1, 40000, "bhsd", True, None),
    (16, 32, 8, 2100, "batch1", True, "padding"), (2, 32, 1, 9000, "bhsd", True, None), (300, 4, 1, 40, "bhsd", True, None)])
def test_decode_that_accumulates_weights_vs_fp64(B, H, Hkv, S, layout, with_lengths, mask):
    q, k, v, _, lengths, mask, _, used = _tree_case(B, H, Hkv, 1, S, layout, None, with_lengths, mask, seed=S)
    weights = torch.rand(B, Hkv, S + 9, generator=_gen(2)).cuda()
    before = weights.clone()
    out = decode_attn_accumulate(q, k, v, weights, used, mask)
    visible = torch.arange(S, device="cuda")[None, None] <= (torch.tensor(lengths, device="cuda") if with_lengths else torch.full((B,), S - 1, device="cuda"))[:, None, None]
    if mask is not None:
        visible = visible & mask[:, 0, :, :S]
    ref, spread, p = _reference(q, k, v, visible)
    _check(out, ref, spread, 1)
    gained = p.view(B, Hkv, H // Hkv, S).sum(2)
    # the sum's own rounding (2^-24 of it, once for each head), and each probability's: scores of up to a hundred
    # in fp32 products and one fp32 exponential argument, 2^-17, exponential and inverse sum 2^-21
    excess = (weights[..., :S].double() - before[..., :S].double() - gained).abs() - (2.0 ** -22 * weights[..., :S].double() + 2.0 ** -16 * gained)
    assert float(excess.max()) <= 0
    assert torch.equal(weights[..., S:], before[..., S:])
    assert torch.equal(weights[..., :S][~visible.expand(B, Hkv, S)], before[..., :S][~visible.expand(B, Hkv, S)])
    again = before.clone()
    assert torch.equal(out, decode_attn_accumulate(q, k, v, again, used, mask)) and torch.equal(again, weights)


def _evict_reference(weights, used, keep, recent):
    """Rows that stay, of one head."""
    if used <= keep:
        return list(range(used))
    w = [float("inf") if x != x else x for x in weights[:used - recent].tolist()]
    nan = [x != x for x in weights[:used - recent].tolist()]
    order = sorted(range(used - recent), key=lambda i: (not nan[i], -w[i], i))[:keep - recent]
    return sorted(order) + list(range(used - recent, used))


@pytest.mark.gpu
@pytest.mark.parametrize("B,Hkv,S,keep,recent,layout,kind", [
    (1, 1, 1, 1, 0, "bhsd", "ties"), (1, 1, 2, 1, 1, "bhsd", "ties"), (2, 2, 100, 33, 7, "bhsd", "ties"), (2, 2, 100, 100, 20, "bshd", "spread"),
    (2, 3, 257, 300, 5, "bhsd", "spread"), (1, 8, 4096, 2048, 512, "bhsd", "spread"), (3, 2, 5000, 1, 0, "bhsd", "equal"), (3, 2, 5000, 77, 77, "sliced", "spread"),
    (2, 2, 2100, 2000, 3, "bhsd", "special"), (1, 1, 70000, 9000, 100, "bhsd", "ties"), (1, 1, 400000, 50, 10, "batch1", "ties"),
    (40, 8, 600, 64, 16, "bhsd", "spread")])
def test_eviction_vs_the_definition(B, Hkv, S, keep, recent, layout, kind):
    k, v = _cache(B, Hkv, S, 1, layout)
    g, rng = _gen(S), random.Random(S)
    w = torch.exp(3 * torch.randn(B, Hkv, S, generator=g))
    if kind == "ties":
        w = (w * 2).round().clamp_max(5) / 4
    elif kind == "equal":
        w[:] = 0.5
    elif kind == "special":
        for value in (float("nan"), float("inf"), float("-inf"), -0.0, 0.0, -1.0, 1e-42, -float("nan")):
            w.view(-1)[torch.randperm(w.numel(), generator=g)[: w.numel() // 12]] = value
    used = [rng.randint(0, S) for _ in range(B)]
    used[0] = S
    if B > 1:
        used[1] = min(S, keep)
    if B > 2:
        used[2] = S + 10 if kind == "equal" else 0
    lengths = torch.tensor(used, dtype=torch.int32, device="cuda")
    weights = w.cuda()
    k2, v2, w2, kept = evict_cache(k, v, weights, keep, recent, lengths)
    assert k2.shape == v2.shape == (B, Hkv, keep, 128) and w2.shape == kept.shape == (B, Hkv, keep)
    for b in range(B):
        for h in range(Hkv):
            rows = _evict_reference(w[b, h], min(used[b], S), keep, recent)
            assert kept[b, h].tolist() == rows + [-1] * (keep - len(rows))
            for got, x in ((k2, k), (v2, v), (w2, weights)):
                assert torch.equal(got[b, h, :len(rows)].nan_to_num(7.0), x[b, h, rows].nan_to_num(7.0)) and not bool(got[b, h, len(rows):].any())
    room = [torch.full((B, Hkv, keep + 3, 128), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)] + [torch.full((B, Hkv, keep + 5), 7.0, device="cuda")]
    again = evict_cache(k, v, weights, keep, recent, lengths, out=room)
    assert all(torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) for a, b in zip(again, (k2, v2, w2, kept)))
    assert all(bool((x[:, :, keep:] == 7).all()) for x in room), "rows behind `keep` are left as they were"


@pytest.mark.gpu
def test_a_serving_step_in_a_graph_and_on_another_stream():
    """Draft tree over two layers' caches, verification, the accepted rows moved, a step that accumulates, eviction - eagerly, on
    a side stream, and captured twice into graphs of one pool that are replayed in turn."""
    B, H, Hkv, n, S, V = 3, 8, 2, 7, 150, 300
    tokens, target, draft, uniform, parents = _verify_case(B, n, V, torch.float32, "random", "sampled", 8)
    tokens, target, draft, uniform = (x.cuda() for x in (tokens, target, draft, uniform))
    up = torch.tensor(parents, dtype=torch.int32, device="cuda")
    start = [x for i in range(2) for x in _cache(B, Hkv, S, i)]
    q, q1 = _queries(B, H, n, 1), _queries(B, H, 1, 2)
    first = torch.tensor([100, 61, 0], dtype=torch.int32, device="cuda")
    base = torch.rand(B, Hkv, S, generator=_gen(4)).cuda()

    def step():
        caches, lengths, weights = [x.clone() for x in start], first.clone(), base.clone()
        outs = [tree_attn(q, caches[i], caches[i + 1], up, lengths) for i in (0, 2)]
        accepted, path, new = verify_drafts(tokens, target, draft, uniform, up)
        keep_drafts(caches, lengths, path)
        lengths += accepted + 1
        outs.append(decode_attn_accumulate(q1, caches[0], caches[1], weights, lengths))
        return outs + [accepted, path, new, weights, *caches, *evict_cache(caches[0], caches[1], weights, 40, 10, lengths + 1)]

    want = step()
    for b in range(B):                                       # the kept rows are what a chain of the accepted tokens would have written
        m, nodes = int(want[3][b]), want[4][b].tolist()
        for i in range(m + 1):
            assert torch.equal(want[7][b, :, int(first[b]) + i], start[0][b, :, int(first[b]) + nodes[i]])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    with torch.cuda.graph(graphs[0]):
        one = step()
    with torch.cuda.graph(graphs[1], pool=graphs[0].pool()):
        two = step()
    for graph, result in ((graphs[0], one), (graphs[1], two), (graphs[0], one)):
        for x in result:
            x.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(result, want))


@pytest.mark.gpu
def test_autograd_learns_of_what_is_written_in_place():
    """A tensor that a graph has saved and one of these calls has overwritten since: backward raises, as behind any in-place operator."""
    k, v = _cache(2, 2, 50, 1)
    q, base = _queries(2, 8, 1, 1), torch.rand(2, 2, 50, generator=_gen(1)).cuda()
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    out = [k.new_zeros(2, 2, 9, 128), k.new_zeros(2, 2, 9, 128), base.new_zeros(2, 2, 9)]
    other = base.clone()
    calls = [(lambda: decode_attn_accumulate(q, k, v, base), [base]), (lambda: keep_drafts([k, v], ints([9, 40]), ints([[0, 2], [1, -1]])), [k, v]),
             (lambda: evict_cache(k, v, other, 7, out=out), out)]
    for call, written in calls:
        for x in written:
            leaf = torch.ones((), device="cuda", dtype=x.dtype, requires_grad=True)
            (leaf * x).sum().backward()
            saved = (leaf * x).sum()
            with torch.no_grad():
                call()
            with pytest.raises(RuntimeError, match="inplace"):
                saved.backward()
    assert other._version == 0
    with torch.inference_mode():                             # whose tensors have no versions
        w = torch.zeros(2, 2, 50, device="cuda")
        decode_attn_accumulate(q, k, v, w)
        keep_drafts([k.clone()], ints([9, 40]), ints([[0, 2], [1, -1]]))


def _calls(q, k, w, probs, tok, u, ints):
    """A call of each operator that takes the given tensors."""
    return [lambda: tree_attn(q, k, k), lambda: decode_attn_accumulate(q[:, :, :1], k, k, w), lambda: verify_drafts(tok, probs, None, u),
            lambda: keep_drafts([k], ints(2), ints(2, 4)), lambda: evict_cache(k, k, w, 5)]


def test_tensors_without_memory_are_refused():
    """Fake tensors, whose addresses are zero and an offset, before any address is looked at."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        q, k, w = torch.zeros(2, 8, 4, 128, dtype=torch.bfloat16, device="cuda"), torch.zeros(2, 2, 60, 128, dtype=torch.bfloat16, device="cuda")[:, :, 10:], torch.zeros(2, 2, 50, device="cuda")
        ints = lambda *shape: torch.zeros(*shape, dtype=torch.int32, device="cuda")
        for call in _calls(q, k, w, torch.ones(2, 4, 9, device="cuda"), torch.zeros(2, 4, dtype=torch.int64, device="cuda"), torch.zeros(2, 4, device="cuda"), ints):
            with pytest.raises(ValueError, match="memory of their own"):
                call()


@pytest.mark.gpu
def test_what_looks_inside_operators_is_refused():
    """Tangents, recorders and batched tensors are not passed by; a subclass that leaves operators alone is a tensor like others."""
    import torch.autograd.forward_ad as fw
    from torch.fx.experimental.proxy_tensor import make_fx
    ints = lambda *shape: torch.zeros(*shape, dtype=torch.int32, device="cuda")
    given = [_queries(2, 8, 4, 1), _cache(2, 2, 50, 1)[0], torch.rand(2, 2, 50, generator=_gen(1)).cuda(), torch.ones(2, 4, 9, device="cuda"),
             torch.zeros(2, 4, dtype=torch.int64, device="cuda"), torch.rand(2, 4, generator=_gen(2)).cuda()]
    with fw.dual_level():
        duals = [x if x.dtype == torch.int64 else fw.make_dual(x, torch.ones_like(x)) for x in given]
        for call in _calls(*duals, ints):
            with pytest.raises(RuntimeError, match="tangents"):
                call()
        for call in _calls(*given, ints):                    # no tangents among these
            call()
    for which in range(5):
        def one(x):
            _calls(x, *given[1:], ints)[0]() if which == 0 else _calls(*given, ints)[which]()
            return x + 1

        with pytest.raises(RuntimeError, match="recorded"):
            torch.jit.trace(one, (given[0],), check_trace=False)
        with pytest.raises(RuntimeError, match="recorded"):
            make_fx(one)(given[0])
    with pytest.raises(RuntimeError):
        torch.vmap(lambda x: tree_attn(x, given[1], given[1]))(given[0][None])

    class Named(torch.Tensor):
        pass

    assert torch.equal(tree_attn(given[0].as_subclass(Named), given[1], given[1]).as_subclass(torch.Tensor), tree_attn(given[0], given[1], given[1]))
    assert torch.equal(tree_attn(torch.nn.Parameter(given[0], requires_grad=False), given[1], given[1]), tree_attn(given[0], given[1], given[1]))


@pytest.mark.gpu
def test_negated_views_keep_their_sign():
    """The imaginary part of a conjugate is a view whose sign is a flag."""
    negated = lambda x: torch.complex(torch.zeros_like(x), -x).conj().imag
    k, w = _cache(2, 2, 50, 1)[0], torch.rand(2, 2, 50, generator=_gen(1)).cuda()
    probs, tok, u = torch.rand(2, 4, 9, generator=_gen(3)).cuda(), torch.randint(9, (2, 4), generator=_gen(4)).cuda(), torch.rand(2, 4, generator=_gen(2)).cuda()
    assert negated(w).is_neg() and torch.equal(negated(w), w)
    want = verify_drafts(tok, probs, probs.flip(-1), u)
    for got in (verify_drafts(tok, negated(probs), probs.flip(-1), u), verify_drafts(tok, probs, negated(probs.flip(-1)), u), verify_drafts(tok, probs, probs.flip(-1), negated(u))):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(torch.equal(a, b) for a, b in zip(evict_cache(k, k, negated(w), 9, 3), evict_cache(k, k, w, 9, 3)))
    with pytest.raises(ValueError, match="negated"):         # written in place
        decode_attn_accumulate(_queries(2, 8, 1, 1), k, k, negated(w))
    with pytest.raises(ValueError):
        evict_cache(k, k, w, 9, out=(k.new_zeros(2, 2, 9, 128), k.new_zeros(2, 2, 9, 128), negated(w)))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 4, 20])
def test_rows_at_odd_addresses_are_copied(n):
    """Contiguous tensors that begin between two 16-byte boundaries, and a batch of one whose unused strides are odd."""
    def odd(x):
        room = torch.empty(x.numel() + 8, dtype=x.dtype, device="cuda")[1:x.numel() + 1].view(x.shape)
        return room.copy_(x)

    def strange(x):
        return x.as_strided(x.shape, (3, 5, 128, 1))

    (k, v), q = _cache(1, 1, 70, 2), _queries(1, 4, n, 2)
    w = torch.rand(1, 1, 70, generator=_gen(1)).cuda()
    want, want_cut = tree_attn(q, k, v), evict_cache(k, v, w, 9, 3)
    want_one = decode_attn_accumulate(q[:, :, :1], k, v, w.clone())
    for change in (odd, strange):
        k2, v2 = change(k), change(v)
        q2 = odd(q)
        assert q2.is_contiguous() and k2.is_contiguous() and torch.equal(k2, k)
        assert torch.equal(tree_attn(q2, k2, v), want) and torch.equal(tree_attn(q, k, v2), want)
        assert torch.equal(decode_attn_accumulate(q2[:, :, :1], k2, v2, w.clone()), want_one)
        assert all(torch.equal(a, b) for a, b in zip(evict_cache(k2, v2, w, 9, 3), want_cut))


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hkv,rows", [(32, 8, 4), (32, 32, 1), (36, 2, 32), (8, 1, 8)])
def test_scratch_of_the_step_with_weights(lib, H, Hkv, rows):
    """A score per key and query head (in groups of 16 where a KV head has more), and the partial results: no more."""
    import ctypes
    B, S, need = 16, 65536, ctypes.c_int64(0)
    p = torch.zeros(64, dtype=torch.uint8, device="cuda").data_ptr()
    qs, st = (ctypes.c_int64 * 3)(H * 128, H * 128, 128), (ctypes.c_int64 * 3)(Hkv * S * 128, 128, S * 128)
    rc = lib.intra_b200_decode_accumulate(p, p, p, None, None, p, p, None, 0, need, B, S, H, Hkv, qs, st, st, None, S * Hkv, S, 0.1, 0, None)
    assert rc == 1                                           # nothing is launched
    units = B * Hkv * (1 if rows <= 16 else 2)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert need.value <= 4 * (B * Hkv * rows * S + (units + 2 * sms) * 16 * 130)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_refusals(device):
    bf = lambda *shape: torch.zeros(*shape, dtype=torch.bfloat16, device=device)
    ints = lambda *shape: torch.zeros(*shape, dtype=torch.int32, device=device)
    q, k, w = bf(2, 8, 4, 128), bf(2, 2, 50, 128), torch.zeros(2, 2, 50, device=device)
    probs, tok, u = torch.ones(2, 4, 9, device=device), torch.zeros(2, 4, dtype=torch.int64, device=device), torch.zeros(2, 4, device=device)
    if device == "cpu":                                      # nothing runs without a GPU
        for call in (lambda: tree_attn(q, k, k), lambda: decode_attn_accumulate(q[:, :, :1], k, k, w), lambda: verify_drafts(tok, probs, None, u),
                     lambda: keep_drafts([k], ints(2), ints(2, 4)), lambda: evict_cache(k, k, w, 5)):
            with pytest.raises(ValueError, match="CUDA"):
                call()
        return
    bad = [
        lambda: tree_attn(q.float(), k, k), lambda: tree_attn(q[..., :64], k[..., :64], k[..., :64]), lambda: tree_attn(q, k, k[:, :, :9]),
        lambda: tree_attn(q[:1], k, k), lambda: tree_attn(q[:, :7], k, k), lambda: tree_attn(q, k[:, :, :3], k[:, :, :3]),
        lambda: tree_attn(bf(2, 8, 65, 128), bf(2, 2, 70, 128), bf(2, 2, 70, 128)), lambda: tree_attn(q[:, :, :0], k, k), lambda: tree_attn(q, k[:, :0], k[:, :0]),
        lambda: tree_attn(q, k, k, ints(3)), lambda: tree_attn(q, k, k, ints(4).long()), lambda: tree_attn(q, k, k, None, ints(3)),
        lambda: tree_attn(q, k, k, None, ints(2).cpu()), lambda: tree_attn(q, k, k, None, None, torch.ones(2, 1, 4, 49, dtype=torch.bool, device=device)),
        lambda: tree_attn(q, k, k, None, None, torch.ones(2, 8, 4, 50, dtype=torch.bool, device=device)), lambda: tree_attn(q, k, k, None, None, bf(2, 1, 4, 50)),
        lambda: tree_attn(q, k, k, softmax_scale=0.0), lambda: tree_attn(q, k, k, softmax_scale=float("nan")),
        lambda: decode_attn_accumulate(q, k, k, w), lambda: decode_attn_accumulate(q[:, :, :1], k, k, w[:, :, :49]), lambda: decode_attn_accumulate(q[:, :, :1], k, k, w.half()),
        lambda: decode_attn_accumulate(q[:, :, :1], k, k, w[:, :1].expand(2, 2, 50)), lambda: decode_attn_accumulate(q[:, :, :1], k, k, torch.zeros(2, 2, 100, device=device)[..., ::2]),
        lambda: verify_drafts(tok, probs.double(), None, u), lambda: verify_drafts(tok.float(), probs, None, u), lambda: verify_drafts(tok, probs, probs.half(), u),
        lambda: verify_drafts(tok, probs, probs[:, :2], u), lambda: verify_drafts(tok, probs, None, u.double()), lambda: verify_drafts(tok[:, :3], probs, None, u),
        lambda: verify_drafts(tok, probs, None, u, ints(5)), lambda: verify_drafts(torch.zeros(1, 65, dtype=torch.int64, device=device), torch.ones(1, 65, 3, device=device), None, torch.zeros(1, 65, device=device)),
        lambda: keep_drafts([k, k], ints(2), ints(2, 4)), lambda: keep_drafts([k, k[:, :, 1:]], ints(2), ints(2, 4)), lambda: keep_drafts([k], None, ints(2, 4)),
        lambda: keep_drafts([k[:, :1].expand(2, 2, 50, 128)], ints(2), ints(2, 4)), lambda: keep_drafts([k], ints(2), ints(2, 51)), lambda: keep_drafts([k], ints(2), ints(2, 4).long()),
        lambda: keep_drafts([k], ints(2), ints(2, 0)), lambda: keep_drafts([bf(2, 2, 50, 132)[..., 2:130]], ints(2), ints(2, 4)),
        lambda: evict_cache(k, k, w, 0), lambda: evict_cache(k, k, w, 5, 6), lambda: evict_cache(k, k, w, 5, -1), lambda: evict_cache(k, k, w[:, :, :49], 5),
        lambda: evict_cache(k, k[:, :, :9], w, 5), lambda: evict_cache(k, k, w, 5, out=(k, bf(2, 2, 5, 128), torch.zeros(2, 2, 5, device=device))),
        lambda: evict_cache(k, k, w, 5, out=(bf(2, 2, 4, 128), bf(2, 2, 5, 128), torch.zeros(2, 2, 5, device=device)))]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")
    grad = [lambda: tree_attn(q.clone().requires_grad_(True), k, k), lambda: verify_drafts(tok, probs.clone().requires_grad_(True), None, u),
            lambda: keep_drafts([k.clone().requires_grad_(True)], ints(2), ints(2, 4)), lambda: evict_cache(k, k, w.clone().requires_grad_(True), 5),
            lambda: decode_attn_accumulate(q[:, :, :1], k, k, w.clone().requires_grad_(True))]
    for call in grad:
        with pytest.raises(RuntimeError, match="forward-only"):
            call()


@pytest.mark.gpu
def test_batches_beyond_a_launch_are_refused():
    """65,535 heads with weights, 65,535 sequences with a mask; one more is an error, and without a mask it runs."""
    B = 65536
    x = torch.randn(1, 1, 17, 128, generator=_gen(1)).to(torch.bfloat16).cuda()
    q, k = x.expand(B, 1, 17, 128), x.expand(B, 1, 17, 128)
    mask = torch.ones(1, 1, 1, 17, dtype=torch.bool, device="cuda").expand(B, 1, 1, 17)
    with pytest.raises(ValueError):
        tree_attn(q, k, k, mask=mask)
    with pytest.raises(ValueError):
        decode_attn_accumulate(q[:, :, :1], k, k, torch.zeros(B, 1, 17, device="cuda"))
    out = tree_attn(q, k, k)
    assert torch.equal(out, out[:1].expand_as(out)) and torch.equal(out[:1], tree_attn(x, x, x))


@pytest.mark.gpu
def test_empty_batches():
    k, w = torch.zeros(0, 2, 50, 128, dtype=torch.bfloat16, device="cuda"), torch.zeros(0, 2, 50, device="cuda")
    q = torch.zeros(0, 8, 4, 128, dtype=torch.bfloat16, device="cuda")
    assert tree_attn(q, k, k).shape == (0, 4, 8, 128)
    assert decode_attn_accumulate(q[:, :, :1], k, k, w).shape == (0, 1, 8, 128)
    probs = torch.zeros(0, 4, 9, device="cuda")
    assert [x.shape for x in verify_drafts(probs[..., 0].long(), probs, None, probs[..., 0])] == [(0,), (0, 4), (0, 4)]
    empty = torch.zeros(0, 4, dtype=torch.int32, device="cuda")
    keep_drafts([k], empty[:, 0], empty)
    assert evict_cache(k, k, w, 5)[3].shape == (0, 2, 5)


def test_c_entries_reject_bad_arguments_without_a_gpu(lib):
    """Status codes, before any GPU is touched."""
    import ctypes
    buf = torch.zeros(4096, dtype=torch.uint8)
    p, st, need = buf.data_ptr(), (ctypes.c_int64 * 3)(1024, 128, 128), ctypes.c_int64(0)
    odd = (ctypes.c_int64 * 3)(1024, 4, 128)

    def tree(q=p, n=4, S=8, H=2, Hkv=1, scale=0.1, qs=st, ms=None, mask=None):
        return lib.intra_b200_tree_attn(q, p, p, None, None, mask, p, None, 0, need, 1, S, H, Hkv, n, qs, st, st, 0, 0, ms, scale, 0, None)

    assert tree(q=None) == tree(n=0) == tree(n=9) == tree(H=3, Hkv=2) == tree(scale=0.0) == tree(mask=p) == -1
    assert tree(n=65, S=70) == -2 and tree(q=p + 2) == tree(qs=odd) == -3

    def decode(w=p, qs=st, ws=8, B=1, scale=0.1):
        return lib.intra_b200_decode_accumulate(p, p, p, None, None, p, w, None, 0, need, B, 8, 2, 1, qs, st, st, None, ws, 8, scale, 0, None)

    assert decode(w=None) == decode(B=0) == decode(B=2, ws=0) == decode(scale=-1.0) == -1 and decode(w=p + 2) == decode(qs=odd) == -3

    def verify(t=p, n=4, V=9, kind=0, ts=st):
        return lib.intra_b200_verify_drafts(p, 1, t, None, kind, p, None, p, p, p, 1, n, V, ts, None, 4, 4, 0, 0, None)

    assert verify(t=None) == verify(n=0) == verify(V=0) == verify(kind=3) == verify(ts=None) == -1 and verify(n=65) == verify(V=2 ** 30 + 1) == -2 and verify(t=p + 1) == -3

    def keep(ptrs=(p,), n=4, S=8, s=(1024, 128, 128), step=3):
        return lib.intra_b200_keep_drafts((ctypes.c_void_p * 1)(*ptrs), (ctypes.c_int64 * 3)(*s), step, 1, p, p, 4, 1, S, 1, n, 0, None)

    assert keep(ptrs=(None,)) == keep(n=9) == keep(s=(0, 128, 128)) == keep(step=2) == -1 and keep(n=65, S=70) == -2 and keep(ptrs=(p + 8,)) == -3

    def evict(k=p, keep=4, recent=1, out=st):
        return lib.intra_b200_evict(k, p, p, None, p, p, p, p, 1, 8, 1, keep, recent, st, st, st, out, st, st, 0, None)

    assert evict(k=None) == evict(keep=0) == evict(recent=5) == evict(out=(ctypes.c_int64 * 3)(0, 128, 128)) == -1 and evict(out=odd) == evict(k=p + 2) == -3


@pytest.mark.gpu
@pytest.mark.parametrize("n", [2, 20, 50])
def test_heads_that_share_a_cache_and_masks_that_share_rows(n):
    """KV heads expanded from one (stride 0), a mask expanded over heads and longer than the cache, lengths with a stride."""
    B, H, S = 2, 8, 333
    k, v = _cache(B, 1, S, 5)
    q, k8, v8 = _queries(B, H, n, 5), k.expand(B, 2, S, 128), v.expand(B, 2, S, 128)
    mask = (torch.rand(B, 1, n, S + 20, generator=_gen(6)) < 0.7).cuda().expand(B, H, n, S + 20)
    lengths = torch.tensor([[200, -1], [S - n, -1]], dtype=torch.int32, device="cuda")[:, 0]
    out = tree_attn(q, k8, v8, None, lengths, mask)
    ref, spread, _ = _reference(q, k8, v8, _visible(B, n, S, None, lengths.tolist(), mask))
    _check(out, ref, spread, n * H // 2)
    assert torch.equal(out, tree_attn(q, k8.contiguous(), v8.contiguous(), None, lengths.contiguous(), mask[:, :1].contiguous()))
    one = mask[:1, :, :1]                                    # one row for all sequences and tokens
    out = tree_attn(q, k8, v8, None, lengths, one)
    ref, spread, _ = _reference(q, k8, v8, _visible(B, n, S, None, lengths.tolist(), one.expand(B, H, n, S + 20)))
    _check(out, ref, spread, n * H // 2)


@pytest.mark.gpu
@pytest.mark.parametrize("n,masked", [(4, False), (12, True), (30, False), (60, True)])
def test_rows_that_are_not_finite_are_redone_for_those_that_see_them(n, masked):
    """Values that are not finite, seen by some tokens and not by others, in pieces of several CTAs: finite rows as they would be
    without, the others what the sum over the visible keys gives."""
    B, H, Hkv, S = 2, 8, 2, 2600
    k, v = _cache(B, Hkv, S, 7)
    q, parents = _queries(B, H, n, 7), [[-1] + [0] * (n - 1)] * B
    lengths = [S - n, 1500]
    up, used = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (parents, lengths))
    mask = torch.ones(B, 1, n, S, dtype=torch.bool, device="cuda")
    bad = {}                                                 # (sequence, token) -> the columns and what they become
    v2 = v.clone()
    v2[0, :, lengths[0] + n - 1, 5] = float("inf")           # the last token's own key: the others are its siblings
    bad[0, n - 1] = (5, float("inf"))
    if masked:
        mask[1, 0, 1:, 700] = False                          # a key of the context that only the first token sees
        v2[1, :, 700, 64:] = float("nan")
        bad[1, 0] = (slice(64, 128), float("nan"))
    given = mask if masked else None
    out = tree_attn(q, k, v2, up, used, given)
    ref, spread, _ = _reference(q, k, v, _visible(B, n, S, parents, lengths, given))
    fixed = out.clone()
    for (b, i), (columns, value) in bad.items():
        got = out[b, i, :, columns]
        assert bool(got.isnan().all()) if value != value else bool((got == value).all())
        fixed[b, i, :, columns] = ref[b, i, :, columns].to(torch.bfloat16)
    _check(fixed, ref, spread, n * H // Hkv)


@pytest.mark.gpu
def test_calls_on_two_streams_at_once(lib):
    """Every operator on two streams whose work overlaps gives what it gives alone, and no kernel gave up a wait."""
    from tests._util import device_status
    cases = [_tree_case(*case, seed=i) for i, case in enumerate([(4, 32, 8, 30, 3000, "bhsd", "random", True, "random"), (4, 32, 8, 60, 2000, "bhsd", "random", True, None),
                                                                 (8, 32, 8, 4, 3000, "bhsd", "random", True, None)])]
    tokens, target, draft, uniform, _ = (x if x is None else x.cuda() for x in _verify_case(16, 6, 5000, torch.float32, None, "sampled", 2))
    k, v = _cache(4, 8, 4000, 3)
    q1, base = _queries(4, 32, 1, 3), torch.rand(4, 8, 4000, generator=_gen(3)).cuda()

    def calls():
        weights = base.clone()
        outs = [tree_attn(q, kk, vv, up, used, mask) for q, kk, vv, _, _, mask, up, used in cases]
        outs += [*verify_drafts(tokens, target, draft, uniform), decode_attn_accumulate(q1, k, v, weights), *evict_cache(k, v, weights, 500, 100)]
        return outs

    want = calls()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for stream, results in zip(streams, got):
            with torch.cuda.stream(stream):
                results.append(calls())
    torch.cuda.synchronize()
    for results in got:
        for result in results:
            assert all(torch.equal(a, b) for a, b in zip(result, want))
    assert device_status(lib) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["tree", "tree rows", "verify", "keep", "decode", "evict"])
def test_the_first_call_of_a_process_may_be_captured(name):
    code = f"""
import torch
from intra_b200 import decode_attn_accumulate, evict_cache, keep_drafts, tree_attn, verify_drafts
name = {name!r}
g = torch.Generator(device="cuda").manual_seed(1)
q, k, v = (torch.randn(2, h, s, 128, device="cuda", generator=g).bfloat16() for h, s in ((8, 20), (2, 300), (2, 300)))
w, p, u = (torch.rand(*s, device="cuda", generator=g) for s in ((2, 2, 300), (2, 3, 50), (2, 3)))
t = torch.randint(50, (2, 3), device="cuda", generator=g)
used, path = torch.tensor([100, 200], dtype=torch.int32, device="cuda"), torch.tensor([[0, 2, 5], [0, 1, -1]], dtype=torch.int32, device="cuda")
def call():
    cache, weights = k.clone(), w.clone()
    if name.startswith("tree"):
        return [tree_attn(q if "rows" in name else q[:, :, :2], k, v)]
    if name == "verify":
        return verify_drafts(t, p, None, u)
    if name == "keep":
        keep_drafts([cache], used, path)
        return [cache]
    if name == "decode":
        return [decode_attn_accumulate(q[:, :, :1], k, v, weights), weights]
    return evict_cache(k, v, w, 40, 10)
stream = torch.cuda.Stream()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=stream):
    got = call()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, call()))
print("same")
"""
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert out.returncode == 0 and out.stdout.strip() == "same", out.stdout + out.stderr


@pytest.mark.gpu
def test_latency_table_of_the_serving_operators(tmp_path):
    """`python -m intra_b200.bench_kernel serve` runs them one after the other, and alone."""
    path = tmp_path / "rows.json"
    out = subprocess.run([sys.executable, "-m", "intra_b200.bench_kernel", "serve", "--seqlens", "70,700", "--batch", "2", "--layers", "3", "--drafts", "6",
                          "--vocab", "1000", "--iters", "2", "--warmup", "1", "--out", str(path)], capture_output=True, text=True, timeout=600, cwd=ROOT)
    assert out.returncode == 0, out.stdout[-2000:] + out.stderr[-2000:]
    rows = json.loads(path.read_text())["rows"]
    assert [r["seqlen"] for r in rows] == [70, 700]
    for r in rows:
        assert {"dense", "tree", "verify", "keep", "step", "decode", "decode_weights", "evict", "tree_gbs"} <= set(r) and min(r.values()) > 0


def test_interleaved_caches_are_told_from_overlapping_ones():
    from intra_b200.serving import _overlapping
    packed = torch.zeros(3, 50, 2, 4, 128, dtype=torch.bfloat16)                 # (batch, row, K or V, head, 128)
    k, v = packed[:, :, 0].transpose(1, 2), packed[:, :, 1].transpose(1, 2)
    assert not _overlapping([k, v]) and _overlapping([k, k]) and _overlapping([k, v, v])
    flat = packed.view(-1)
    for shift in (1, 64, 128, 511, 512, 1024, 1025, 50 * 1024 - 512):
        other = flat[shift:].as_strided((2, 4, 30, 128), k.stride())
        first = flat.as_strided((2, 4, 30, 128), k.stride())
        mine, theirs = (set((x.storage_offset() + torch.arange(2)[:, None, None, None] * k.stride(0) + torch.arange(4)[:, None, None] * k.stride(1)
                             + torch.arange(30)[:, None] * k.stride(2) + torch.arange(128)).flatten().tolist()) for x in (first, other))
        assert _overlapping([first, other]) == _overlapping([other, first]) == bool(mine & theirs), shift
    assert _overlapping([v, packed[:, :, 1].transpose(1, 2)]) and not _overlapping([packed[0], packed[1], packed[2]])


def test_public_names():
    for name in ("tree_attn", "verify_drafts", "keep_drafts", "decode_attn_accumulate", "evict_cache"):
        assert name in intra_b200.__all__ and callable(getattr(intra_b200, name))
