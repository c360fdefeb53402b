"""What a server does between two tokens of an answer, on the same static caches (batch, KV heads, rows, 128) as the
decode step: attention of drafted tokens, their verification, the accepted rows moved together; a decode step that
accumulates the attention each key receives, and eviction by it.

    out = tree_attn(q, k, v, parents, lengths)                   # per layer: the last token and its drafts, a tree
    accepted, path, tokens = verify_drafts(drafts, target_probs, draft_probs, uniform, parents)
    keep_drafts([k0, v0, k1, v1, ...], lengths, path)            # all layers at once
    lengths += accepted + 1                                      # next: tokens[b, accepted[b]]

    out = decode_attn_accumulate(q, k, v, weights, lengths)      # per layer
    k, v, weights, rows = evict_cache(k, v, weights, keep=2048, recent=256, lengths=lengths)

Node 0 of a tree is the token sampled last; `parents` names for each node the one it follows. None of these has a counterpart in
the reference, whose decode step is one dense token at a time (experiments/llm/intra_token_attn.py:112-134).
Forward only; nothing synchronises, nothing is remembered between calls, every call runs on the current stream.
"""
from __future__ import annotations

import ctypes

import torch

from . import _loader
from ._loader import lib
from .interface import _byte_span, _c_strides, _raise, _raw_stream

MAX_TOKENS = 64             # nodes of a tree: ancestors are kept as 64 bits
_PROB_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _no_grad(*tensors):
    if torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in tensors):
        raise RuntimeError("INTRA kernels are forward-only; call them under torch.no_grad()")


def _rows_usable(x):
    """Rows of 128 that the kernels can read in place."""
    s = x.stride()
    return s[3] == 1 and not (s[0] | s[1] | s[2]) & 7 and not x.data_ptr() & 15


def _attention_inputs(q, k, v):
    """Checks of q (B, H, n, 128) and a cache k, v (B, Hkv, S, 128); tensors whose rows are not 16-byte aligned are copied."""
    for x in (q, k, v):
        if not x.is_cuda or x.dtype != torch.bfloat16 or x.dim() != 4 or x.shape[-1] != 128:
            raise ValueError("INTRA kernels need CUDA bfloat16 tensors (batch, heads, tokens, 128)")
    _no_grad(q, k, v)
    if k.shape != v.shape or k.shape[0] != q.shape[0] or k.shape[1] == 0 or q.shape[1] == 0 or q.shape[1] % k.shape[1]:
        raise ValueError(f"incompatible shapes q={tuple(q.shape)} k={tuple(k.shape)} v={tuple(v.shape)}")
    if k.device != q.device or v.device != q.device:
        raise ValueError("q, k, v must be on the same device")
    return [x if _rows_usable(x) else x.contiguous() for x in (q, k, v)]


def _integers(x, name, shapes, device):
    """An int32 tensor of one of `shapes` on `device`, unit stride in the last dimension."""
    if x is None:
        return None
    if x.dtype != torch.int32 or tuple(x.shape) not in shapes or x.device != device:
        raise ValueError(f"{name} must be int32 of shape {' or '.join(map(str, shapes))} on {device}, got {x.dtype} {tuple(x.shape)} on {x.device}")
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


def _mask(mask, B, n, S, device):
    """(tensor, strides {batch, token, key}) of a boolean mask (B or 1, 1, n or 1, >= S)."""
    if (mask.dtype != torch.bool or mask.dim() != 4 or mask.device != device or mask.shape[0] not in (1, B)
            or mask.shape[2] not in (1, n) or mask.shape[3] < S or (mask.shape[1] != 1 and mask.stride(1) != 0)):
        raise ValueError(f"mask must be bool (batch or 1, 1, tokens or 1, at least {S}) on {device}, the same for every head")
    st = mask.stride()
    return _c_strides(st[0] if mask.shape[0] > 1 else 0, st[2] if mask.shape[2] > 1 else 0, st[3])


def _bsh(x):
    """Strides {batch, token, head} of a (B, heads, tokens, 128) tensor."""
    s = x.stride()
    return _c_strides(s[0], s[2], s[1])


def _ptr(x):
    return None if x is None else x.data_ptr()


def _with_scratch(call, device):
    """Runs call(scratch pointer, its bytes, where the bytes wanted are stored) with a buffer as large as it asks for."""
    need = ctypes.c_int64(0)
    rc = call(None, 0, need)
    if rc == _loader.NEED_SCRATCH:
        scratch = torch.empty(need.value, dtype=torch.uint8, device=device)
        rc = call(scratch.data_ptr(), need.value, need)
    if rc != 0:
        _raise(rc)


def tree_attn(q, k, v, parents=None, lengths=None, mask=None, softmax_scale=None):
    """Attention of n new tokens per sequence, drafts that form a tree, over the cache that holds their keys already.

    q (B, H, n, 128), 1 <= n <= 64; k, v (B, Hkv, S, 128), H a multiple of Hkv. The tokens' own keys are rows lengths[b] ..
    lengths[b] + n - 1; `lengths` (B,) int32 on the GPU, None: the cache's last n rows. (Values that leave the tokens no room
    in the cache are brought into 0 .. S - n; they cannot be refused without a synchronisation.) Token i sees all keys
    before those, its ancestors and itself: parents (n,) or (B, n) int32, parents[i] the earlier token that token i follows, negative for
    none; None: token i follows token i - 1. `mask`, bool (B or 1, 1, n or 1, >= S), hides further keys. Returns (B, n, H, 128)."""
    return _tree(q, k, v, parents, lengths, mask, softmax_scale, False)


def _tree(q, k, v, parents, lengths, mask, softmax_scale, all_own):
    """tree_attn; with `all_own` the tokens see all their own keys, so that the mask decides alone."""
    q, k, v = _attention_inputs(q, k, v)
    B, H, n, D = q.shape
    Hkv, S = k.shape[1:3]
    if not 1 <= n <= MAX_TOKENS or n > S:
        raise ValueError(f"expected 1 to {MAX_TOKENS} tokens whose keys are in the cache, got {n} and a cache of {S} rows")
    dev = q.device
    parents = _integers(parents, "parents", ((n,), (B, n)), dev)
    lengths = _integers(lengths, "lengths", ((B,),), dev)
    m_strides = None if mask is None else _mask(mask, B, n, S, dev)
    out = torch.empty((B, n, H, D), dtype=q.dtype, device=dev)
    if B == 0:
        return out
    scale = 0.08838834764831845 if softmax_scale is None else float(softmax_scale)
    up = parents.stride(0) if parents is not None and parents.dim() == 2 else 0
    qs, ks, vs, stream = _bsh(q), _bsh(k), _bsh(v), _raw_stream(dev.index)

    def call(scratch, nbytes, need):
        return lib.intra_b200_tree_attn(q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(parents), _ptr(lengths), _ptr(mask),
                                        out.data_ptr(), scratch, nbytes, need, B, S, H, Hkv, n, qs, ks, vs, up, all_own, m_strides, scale,
                                        dev.index, stream)

    _with_scratch(call, dev)
    return out


def decode_attn_accumulate(q, k, v, weights, lengths=None, mask=None, softmax_scale=None):
    """Dense attention of one token per sequence, q (B, H, 1, 128), over its cache k, v (B, Hkv, S, 128), that adds to
    `weights`, (B, Hkv, >= S) float32, the probability each key receives, summed over the query heads of its KV head. The token
    sees rows 0 .. lengths[b], its own being the last of them; `lengths` (B,) int32, None: all S. (Values outside 0 ..
    S - 1 are brought into that range.) `mask`, bool (B or 1, 1, 1, >= S), hides further keys. Weights of keys the
    token does not see stay as they are. Returns (B, 1, H, 128)."""
    q, k, v = _attention_inputs(q, k, v)
    B, H, n, D = q.shape
    Hkv, S = k.shape[1:3]
    if n != 1 or S == 0:
        raise ValueError(f"expected one token per sequence and a cache that holds it, got {n} and {S} rows")
    dev = q.device
    if (not weights.is_cuda or weights.dtype != torch.float32 or weights.dim() != 3 or weights.shape[:2] != k.shape[:2]
            or weights.shape[2] < S or weights.device != dev):
        raise ValueError(f"weights must be float32 (batch, KV heads, at least {S}) on {dev}")
    _no_grad(weights)
    _distinct_rows(weights, "weights")
    lengths = _integers(lengths, "lengths", ((B,),), dev)
    m_strides = None if mask is None else _mask(mask, B, 1, S, dev)
    out = torch.empty((B, 1, H, D), dtype=q.dtype, device=dev)
    if B == 0:
        return out
    if mask is not None:
        m_strides = _c_strides(m_strides[0], m_strides[2], 0)
    scale = 0.08838834764831845 if softmax_scale is None else float(softmax_scale)
    qs, ks, vs, stream, ws = _bsh(q), _bsh(k), _bsh(v), _raw_stream(dev.index), weights.stride()

    def call(scratch, nbytes, need):
        return lib.intra_b200_decode_accumulate(q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(mask), _ptr(lengths), out.data_ptr(),
                                                weights.data_ptr(), scratch, nbytes, need, B, S, H, Hkv, qs, ks, vs, m_strides,
                                                ws[0], ws[1], scale, dev.index, stream)

    _with_scratch(call, dev)
    return out


def _distinct_rows(x, name):
    """A tensor that is written needs unit stride in its last dimension and rows that do not share memory."""
    if x.stride(-1) != 1 and x.shape[-1] > 1:
        raise ValueError(f"{name} needs unit stride in the last dimension")
    reach = x.shape[-1]
    for size, stride in sorted(((n, s) for n, s in zip(x.shape[:-1], x.stride()[:-1]) if n > 1), key=lambda d: d[1]):
        if stride < reach:
            raise ValueError(f"{name} has rows that share memory")
        reach = stride * (size - 1) + reach


def verify_drafts(tokens, target_probs, draft_probs, uniform, parents=None):
    """Which drafted tokens the target model accepts, and one token more, so that tokens come out distributed as the target's.

    tokens (B, n) int64 or int32, 1 <= n <= 64: node 0 is the token sampled last, nodes 1 .. n - 1 are drafts. target_probs
    (B, n, V): the target's distribution behind each node; draft_probs (B, n or n - 1, V), of the same type (float32,
    bfloat16 or float16): the distribution the children of each node were drawn from, None for drafts that were not drawn (each counts
    as certain). uniform (B, n) float32 in [0, 1): entry i decides node i, entry 0 draws the last token. parents (n,) or
    (B, n) int32: the node each follows, an earlier one; None: a chain.

    From node 0 on, the children x of the current node are tried in index order: accepted iff uniform * q(x) * Z < R(x), with R the
    target's distribution and Z = 1 at first; a rejection replaces R by max(R / Z - q, 0) and Z by its sum (unless that is
    zero). When none is left the last token is drawn from R: the smallest t with R(0) + .. + R(t) > uniform * sum R. Sums
    and comparisons are in 64 bits.

    Returns accepted (B,) int32, the number m of accepted drafts; path (B, n) int32, the nodes from 0 on, then -1; and tokens
    (B, n) int64: the m accepted ones, the drawn one, then -1. Drafts outside the vocabulary are rejected."""
    if target_probs.dim() != 3 or target_probs.dtype not in _PROB_TYPES or not target_probs.is_cuda:
        raise ValueError("target_probs must be a CUDA float32, bfloat16 or float16 tensor (batch, nodes, vocabulary)")
    B, n, V = target_probs.shape
    dev = target_probs.device
    _no_grad(target_probs, draft_probs, uniform)
    if not 1 <= n <= MAX_TOKENS or V == 0:
        raise ValueError(f"expected 1 to {MAX_TOKENS} nodes and a vocabulary, got {n} and {V}")
    if tokens.dtype not in (torch.int64, torch.int32) or tokens.shape != (B, n) or tokens.device != dev:
        raise ValueError(f"tokens must be int64 or int32 ({B}, {n}) on {dev}")
    if uniform.dtype != torch.float32 or uniform.shape != (B, n) or uniform.device != dev:
        raise ValueError(f"uniform must be float32 ({B}, {n}) on {dev}")
    if draft_probs is not None and (draft_probs.dtype != target_probs.dtype or draft_probs.dim() != 3 or draft_probs.shape[0] != B
                                    or draft_probs.shape[1] not in (n - 1, n) or draft_probs.shape[2] != V or draft_probs.device != dev):
        raise ValueError(f"draft_probs must be {target_probs.dtype} ({B}, {n - 1} or {n}, {V}) on {dev}")
    parents = _integers(parents, "parents", ((n,), (B, n)), dev)
    accepted = torch.empty(B, dtype=torch.int32, device=dev)
    path = torch.empty((B, n), dtype=torch.int32, device=dev)
    out = torch.empty((B, n), dtype=torch.int64, device=dev)
    if B == 0:
        return accepted, path, out
    target_probs, tokens, uniform = (x if x.stride(-1) == 1 else x.contiguous() for x in (target_probs, tokens, uniform))
    if draft_probs is not None and (draft_probs.numel() == 0 or draft_probs.stride(-1) != 1):
        draft_probs = None if draft_probs.numel() == 0 else draft_probs.contiguous()
    up = parents.stride(0) if parents is not None and parents.dim() == 2 else 0
    rc = lib.intra_b200_verify_drafts(tokens.data_ptr(), tokens.dtype == torch.int64, target_probs.data_ptr(), _ptr(draft_probs),
                                      _PROB_TYPES[target_probs.dtype], uniform.data_ptr(), _ptr(parents), accepted.data_ptr(),
                                      path.data_ptr(), out.data_ptr(), B, n, V, _c_strides(*target_probs.stride()),
                                      None if draft_probs is None else _c_strides(*draft_probs.stride()), tokens.stride(0),
                                      uniform.stride(0), up, dev.index, _raw_stream(dev.index))
    if rc != 0:
        _raise(rc)
    return accepted, path, out


def _meet(distance, dims):
    """Does sum a_i * stride_i = distance have a solution with |a_i| < size_i? dims: (size, stride), the largest stride first, each at
    least as large as all that the smaller ones reach."""
    if not dims:
        return distance == 0
    size, stride = dims[0]
    nearest = distance // stride
    return any(-size < a < size and _meet(distance - a * stride, dims[1:]) for a in (nearest, nearest + 1))


def _overlapping(tensors):
    """Do two of these tensors share memory? By their byte ranges, and, where those overlap and the layouts are alike - K and V
    interleaved in one buffer - by their elements."""
    spans = sorted(((*_byte_span(x), i) for i, x in enumerate(tensors)))
    for i, (_, end, a) in enumerate(spans):
        for start, _, b in spans[i + 1:]:
            if start >= end:
                break
            x, y = tensors[a], tensors[b]
            if x.shape != y.shape or x.stride() != y.stride() or x.dtype != y.dtype:
                return True
            dims = sorted(((n, s) for n, s in zip(x.shape, x.stride()) if n > 1), key=lambda d: -d[1])
            reach = 1
            for n, s in reversed(dims):
                if s < reach:
                    return True
                reach += (n - 1) * s
            if (y.data_ptr() - x.data_ptr()) % x.element_size() or _meet((y.data_ptr() - x.data_ptr()) // x.element_size(), dims):
                return True
    return False


def keep_drafts(caches, lengths, path):
    """Moves the cache rows of accepted tokens together, in place: in each of `caches` (a tensor or a sequence of them, K and V of
    all layers, (B, Hkv, S, 128) bfloat16, all of one shape) row lengths[b] + path[b, i] becomes row lengths[b] + i, for every i with path[b, i] >= 0. lengths (B,) int32: rows before the
    tokens' own, as in `tree_attn`; path (B, n) int32, n <= 64, as `verify_drafts` returns it. Entries outside 0 .. n - 1 move
    nothing, and neither does a sequence whose lengths[b] is not in 0 .. S - n. Other rows stay as they are."""
    caches = [caches] if isinstance(caches, torch.Tensor) else list(caches)
    if not caches:
        return
    first = caches[0]
    dev = first.device
    for x in caches:
        if not x.is_cuda or x.dtype != torch.bfloat16 or x.dim() != 4 or x.shape[-1] != 128:
            raise ValueError("INTRA kernels need CUDA bfloat16 tensors (batch, heads, tokens, 128)")
        if x.shape != first.shape or x.device != dev:
            raise ValueError("caches must agree in shape and device")
        if not _rows_usable(x):
            raise ValueError("caches need unit stride in the last dimension and 16-byte aligned rows")
        _distinct_rows(x, "a cache")
    _no_grad(*caches)
    B, Hkv, S, _ = first.shape
    if path.dim() != 2 or not 1 <= path.shape[1] <= min(MAX_TOKENS, S):
        raise ValueError(f"path must be (batch, n) with n from 1 to {min(MAX_TOKENS, S)}")
    path = _integers(path, "path", ((B, path.shape[1]),), dev)
    lengths = _integers(lengths, "lengths", ((B,),), dev)
    if lengths is None:
        raise ValueError("lengths is needed")
    if len(caches) > 1 and _overlapping(caches):
        raise ValueError("caches must not overlap")
    if B == 0 or Hkv == 0:
        return
    pointers = (ctypes.c_void_p * len(caches))(*[x.data_ptr() for x in caches])
    strides = (ctypes.c_int64 * (3 * len(caches)))()
    for i, x in enumerate(caches):
        s = x.stride()
        strides[3 * i:3 * i + 3] = [s[d] if x.shape[d] > 1 else 8 for d in (0, 2, 1)]
    rc = lib.intra_b200_keep_drafts(pointers, strides, len(caches), lengths.data_ptr(), path.data_ptr(), path.stride(0), B, S, Hkv,
                                    path.shape[1], dev.index, _raw_stream(dev.index))
    if rc != 0:
        _raise(rc)


def evict_cache(k, v, weights, keep, recent=0, lengths=None, out=None):
    """Cuts a cache k, v (B, Hkv, S, 128) down to `keep` rows per head: the last `recent` in use and the heaviest of the others by
    `weights` (B, Hkv, >= S) float32, as `decode_attn_accumulate` leaves them, in their order; ties go to the lower row, NaN counts as
    the heaviest. lengths (B,) int32: rows in use, None: all S (values outside 0 .. S are brought into that range). A sequence with no
    more than `keep` rows keeps them all.

    Returns (k, v, weights, kept): the kept rows, their weights and their old places (B, Hkv, keep) int32. Behind a sequence's
    last row come zeros, and -1 in `kept`; lengths are min(lengths, keep) from then on. `out` = (k, v, weights) writes into the
    caller's tensors of at least `keep` rows, whose rows from `keep` on stay as they are; they must not overlap the inputs."""
    for x in (k, v):
        if not x.is_cuda or x.dtype != torch.bfloat16 or x.dim() != 4 or x.shape[-1] != 128:
            raise ValueError("INTRA kernels need CUDA bfloat16 tensors (batch, heads, tokens, 128)")
    _no_grad(k, v, weights)
    B, Hkv, S, D = k.shape
    dev = k.device
    if v.shape != k.shape or v.device != dev or S == 0:
        raise ValueError(f"incompatible shapes k={tuple(k.shape)} v={tuple(v.shape)}")
    if weights.dtype != torch.float32 or weights.dim() != 3 or weights.shape[:2] != k.shape[:2] or weights.shape[2] < S or weights.device != dev:
        raise ValueError(f"weights must be float32 (batch, KV heads, at least {S}) on {dev}")
    keep, recent = int(keep), int(recent)
    if not 1 <= keep or not 0 <= recent <= keep:
        raise ValueError(f"expected keep >= 1 and recent from 0 to keep, got {keep} and {recent}")
    lengths = _integers(lengths, "lengths", ((B,),), dev)
    k, v = (x if _rows_usable(x) else x.contiguous() for x in (k, v))
    weights = weights if weights.stride(-1) == 1 else weights.contiguous()
    if out is None:
        k2, v2 = (torch.empty((B, Hkv, keep, D), dtype=k.dtype, device=dev) for _ in range(2))
        w2 = torch.empty((B, Hkv, keep), dtype=torch.float32, device=dev)
    else:
        k2, v2, w2 = out
        for x in (k2, v2):
            if x.dtype != k.dtype or x.dim() != 4 or x.shape[:2] != k.shape[:2] or x.shape[2] < keep or x.shape[3] != D or x.device != dev:
                raise ValueError(f"out needs bfloat16 ({B}, {Hkv}, at least {keep}, 128) for k and v on {dev}")
            if not _rows_usable(x):
                raise ValueError("out needs unit stride in the last dimension and 16-byte aligned rows")
        if w2.dtype != torch.float32 or w2.dim() != 3 or w2.shape[:2] != k.shape[:2] or w2.shape[2] < keep or w2.device != dev:
            raise ValueError(f"out needs float32 ({B}, {Hkv}, at least {keep}) for the weights on {dev}")
        _no_grad(k2, v2, w2)
        for x in (k2, v2, w2):
            _distinct_rows(x, "out")
        if _overlapping((k2, v2, w2)) or any(_overlapping((x, y)) for x in (k2, v2, w2) for y in (k, v, weights)):
            raise ValueError("out must not overlap the cache: rows are still read while it is written")
    kept = torch.empty((B, Hkv, keep), dtype=torch.int32, device=dev)
    if B == 0 or Hkv == 0:
        return k2[:, :, :keep], v2[:, :, :keep], w2[:, :, :keep], kept
    rc = lib.intra_b200_evict(k.data_ptr(), v.data_ptr(), weights.data_ptr(), _ptr(lengths), k2.data_ptr(), v2.data_ptr(),
                              w2.data_ptr(), kept.data_ptr(), B, S, Hkv, keep, recent, _bsh(k), _bsh(v), _c_strides(*weights.stride()),
                              _written(k2, (0, 2, 1)), _written(v2, (0, 2, 1)), _written(w2, (0, 1)), dev.index, _raw_stream(dev.index))
    if rc != 0:
        _raise(rc)
    return k2[:, :, :keep], v2[:, :, :keep], w2[:, :, :keep], kept


def _written(x, order):
    """Strides of a tensor that is written, those of dimensions of one entry made positive."""
    s = [x.stride(d) if x.shape[d] > 1 else 8 for d in order]
    return _c_strides(s[0], s[1], s[2] if len(s) > 2 else 0)
