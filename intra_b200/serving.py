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
Forward only: gradients, tangents and programs that are being recorded (torch.jit.trace, torch.fx) are refused. Nothing synchronises,
nothing is remembered between calls, every call runs on the current stream; tensors written in place count as modified for autograd.
"""
from __future__ import annotations

import array
import ctypes

import torch
from torch.autograd.graph import increment_version

from . import _loader
from ._loader import lib
from .interface import _byte_span, _c_strides, _dispatch_modes, _forward_ad, _raise, _raw_stream, _tracing_state

MAX_TOKENS = 64             # nodes of a tree: ancestors are kept as 64 bits
_PROB_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_SCALE = 128 ** -0.5


_PLAIN = frozenset((torch.Tensor, torch.nn.Parameter, type(None)))
_tracing = _tracing_state or (lambda: None)
_modes = _dispatch_modes or (lambda: 0)


def _forward_only(*tensors):
    """Refuses what these kernels would pass by without a trace: gradients, tangents, programs that are being recorded, and tensors that
    carry out operators themselves and have no memory of their own (fake or distributed ones). None stands for an argument left out."""
    if not _PLAIN.issuperset(map(type, tensors)):
        for x in tensors:
            if x is not None and type(x).__torch_dispatch__ is not torch.Tensor.__torch_dispatch__:
                raise ValueError(f"INTRA kernels need tensors with memory of their own, not {type(x).__name__}")
    if torch.is_grad_enabled() and True in [x.requires_grad for x in tensors if x is not None]:
        raise RuntimeError("INTRA kernels are forward-only; call them under torch.no_grad()")
    if _tracing() is not None:
        raise RuntimeError("INTRA kernels cannot be recorded by torch.jit.trace")
    if _modes() > 0:
        from torch.fx.experimental.proxy_tensor import get_proxy_mode
        if get_proxy_mode() is not None:
            raise RuntimeError("INTRA kernels cannot be recorded by torch.fx")
    if getattr(_forward_ad, "_current_level", -1) >= 0 and any([x is not None and _forward_ad.unpack_dual(x).tangent is not None for x in tensors]):
        raise RuntimeError("INTRA kernels are forward-only; tangents would be lost")


def _rows_usable(x):
    """Rows of 128 that the kernels can read in place."""
    s = x.stride()
    return s[3] == 1 and not (s[0] | s[1] | s[2]) & 7 and not x.data_ptr() & 15


def _usable(x):
    """x, or a copy whose rows the kernels can read. (contiguous() would hand back a contiguous tensor at an odd address.)"""
    return x if _rows_usable(x) else x.clone(memory_format=torch.contiguous_format)


def _attention_inputs(q, k, v):
    """q (B, H, n, 128) and a cache k, v (B, Hkv, S, 128) as the kernels can read them (tensors whose rows are not 16-byte
    aligned are copied), their strides {batch, token, head} for the C ABI, and their device. Raises for others."""
    bf16, dev, qn, kn = torch.bfloat16, q.device, q.shape, k.shape
    if not (q.is_cuda and q.dtype is bf16 and k.dtype is bf16 and v.dtype is bf16 and len(qn) == 4 and len(kn) == 4
            and qn[3] == 128 and kn[3] == 128):
        raise ValueError("INTRA kernels need CUDA bfloat16 tensors (batch, heads, tokens, 128)")
    if kn != v.shape or kn[0] != qn[0] or kn[1] == 0 or qn[1] == 0 or qn[1] % kn[1]:
        raise ValueError(f"incompatible shapes q={tuple(qn)} k={tuple(kn)} v={tuple(v.shape)}")
    if k.device != dev or v.device != dev:
        raise ValueError("q, k, v must be on the same device")
    qs, ks, vs = q.stride(), k.stride(), v.stride()
    if (qs[3] != 1 or ks[3] != 1 or vs[3] != 1 or (q.data_ptr() | k.data_ptr() | v.data_ptr()) & 15
            or (qs[0] | qs[1] | qs[2] | ks[0] | ks[1] | ks[2] | vs[0] | vs[1] | vs[2]) & 7):
        q, k, v = _usable(q), _usable(k), _usable(v)
        qs, ks, vs = q.stride(), k.stride(), v.stride()
    return (q, k, v, _c_strides(qs[0], qs[2], qs[1]), _c_strides(ks[0], ks[2], ks[1]), _c_strides(vs[0], vs[2], vs[1]), dev)


def _integers(x, name, shape, device, shared=None):
    """An int32 tensor of `shape`, or of shape `shared` that all sequences share, unit stride in the last dimension, and its
    address and batch stride."""
    if x is None:
        return None, None, 0
    n = x.shape
    if x.dtype is not torch.int32 or (n != shape and n != shared) or x.device != device:
        raise ValueError(f"{name} must be int32 of shape {shape}{f' or {shared}' if shared else ''} on {device}, "
                         f"got {x.dtype} {tuple(n)} on {x.device}")
    if x.stride(-1) != 1:
        x = x.contiguous()
    return x, x.data_ptr(), x.stride(0) if len(n) == 2 else 0


def _mask(mask, B, n, S, device):
    """Strides {batch, token, key} of a boolean mask (B or 1, 1, n or 1, >= S)."""
    m = mask.shape
    if (mask.dtype is not torch.bool or len(m) != 4 or mask.device != device or (m[0] != B and m[0] != 1)
            or (m[2] != n and m[2] != 1) or m[3] < S or (m[1] != 1 and mask.stride(1) != 0)):
        raise ValueError(f"mask must be bool (batch or 1, 1, tokens or 1, at least {S}) on {device}, the same for every head")
    st = mask.stride()
    return st[0] if m[0] > 1 else 0, st[2] if m[2] > 1 else 0, st[3]


def _ptr(x):
    return None if x is None else x.data_ptr()


# Bytes of scratch a call wants, by its sizes: asking the library costs as much as a third of a short call.
_SCRATCH = {}
_SCRATCH_MAX = 1024


def _with_scratch(key, call, device):
    """Runs call(scratch pointer, its bytes, where the bytes wanted are stored) with a buffer as large as it asks for."""
    nbytes = _SCRATCH.get(key, 0)
    need = ctypes.c_int64(0)
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    rc = call(_ptr(scratch), nbytes, need)
    if rc == _loader.NEED_SCRATCH:
        if len(_SCRATCH) >= _SCRATCH_MAX:
            _SCRATCH.clear()
        nbytes = _SCRATCH[key] = need.value
        scratch = torch.empty(nbytes, dtype=torch.uint8, device=device)
        rc = call(scratch.data_ptr(), nbytes, need)
    if rc != 0:
        _raise(rc)


def tree_attn(q, k, v, parents=None, lengths=None, mask=None, softmax_scale=None):
    """Attention of n new tokens per sequence, drafts that form a tree, over the cache that holds their keys already.

    q (B, H, n, 128), 1 <= n <= 64; k, v (B, Hkv, S, 128), H a multiple of Hkv. The tokens' own keys are rows lengths[b] ..
    lengths[b] + n - 1; `lengths` (B,) int32 on the GPU, None: the cache's last n rows. (Values that leave the tokens no room
    in the cache are brought into 0 .. S - n; they cannot be refused without a synchronisation.) Token i sees all keys
    before those, its ancestors and itself: parents (n,) or (B, n) int32, parents[i] the earlier token that token i follows,
    negative for none; None: token i follows token i - 1. `mask`, bool (B or 1, 1, n or 1, >= S), hides further keys.
    Returns (B, n, H, 128); a token that sees nothing gets zeros."""
    return _tree(q, k, v, parents, lengths, mask, softmax_scale, False)


def _tree(q, k, v, parents, lengths, mask, softmax_scale, all_own):
    """tree_attn; with `all_own` the tokens see all their own keys, so that the mask decides alone."""
    _forward_only(q, k, v, parents, lengths, mask)
    q, k, v, qs, ks, vs, dev = _attention_inputs(q, k, v)
    B, H, n, D = q.shape
    _, Hkv, S, _ = k.shape
    if not 1 <= n <= MAX_TOKENS or n > S:
        raise ValueError(f"expected 1 to {MAX_TOKENS} tokens whose keys are in the cache, got {n} and a cache of {S} rows")
    parents, up, up_stride = _integers(parents, "parents", (B, n), dev, (n,))
    lengths, used, _ = _integers(lengths, "lengths", (B,), dev)
    ms = None if mask is None else _c_strides(*_mask(mask, B, n, S, dev))
    out = q.new_empty((B, n, H, D))
    if B == 0:
        return out
    index, scale = dev.index, _SCALE if softmax_scale is None else float(softmax_scale)
    stream = _raw_stream(index)

    def call(scratch, nbytes, need):
        return lib.intra_b200_tree_attn(q.data_ptr(), k.data_ptr(), v.data_ptr(), up, used, _ptr(mask), out.data_ptr(), scratch,
                                        nbytes, need, B, S, H, Hkv, n, qs, ks, vs, up_stride, all_own, ms, scale, index, stream)

    _with_scratch((n, B, S, H, Hkv, ms is None, index), call, dev)
    return out


def decode_attn_accumulate(q, k, v, weights, lengths=None, mask=None, softmax_scale=None):
    """Dense attention of one token per sequence, q (B, H, 1, 128), over its cache k, v (B, Hkv, S, 128), that adds to
    `weights`, (B, Hkv, >= S) float32, the probability each key receives, summed over the query heads of its KV head. The token
    sees rows 0 .. lengths[b], its own being the last of them; `lengths` (B,) int32, None: all S. (Values outside 0 ..
    S - 1 are brought into that range.) `mask`, bool (B or 1, 1, 1, >= S), hides further keys. Weights of keys the
    token does not see stay as they are. Returns (B, 1, H, 128)."""
    _forward_only(q, k, v, weights, lengths, mask)
    q, k, v, qs, ks, vs, dev = _attention_inputs(q, k, v)
    B, H, n, D = q.shape
    _, Hkv, S, _ = k.shape
    if n != 1 or S == 0:
        raise ValueError(f"expected one token per sequence and a cache that holds it, got {n} and {S} rows")
    wn, ws = weights.shape, weights.stride()
    if weights.dtype is not torch.float32 or len(wn) != 3 or wn[0] != B or wn[1] != Hkv or wn[2] < S or weights.device != dev:
        raise ValueError(f"weights must be float32 (batch, KV heads, at least {S}) on {dev}")
    if weights.is_neg():
        raise ValueError("weights must not be a negated view")
    if not (ws[2] == 1 and ws[1] >= wn[2] and ws[0] >= ws[1] * Hkv):     # else look closer
        _distinct_rows(wn, ws, "weights")
    lengths, used, _ = _integers(lengths, "lengths", (B,), dev)
    ms = None
    if mask is not None:
        ms = _mask(mask, B, 1, S, dev)
        ms = _c_strides(ms[0], ms[2], 0)
    out = q.new_empty((B, 1, H, D))
    if B == 0:
        return out
    index, scale = dev.index, _SCALE if softmax_scale is None else float(softmax_scale)
    stream = _raw_stream(index)

    def call(scratch, nbytes, need):
        return lib.intra_b200_decode_accumulate(q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(mask), used, out.data_ptr(),
                                                weights.data_ptr(), scratch, nbytes, need, B, S, H, Hkv, qs, ks, vs, ms,
                                                ws[0], ws[1], scale, index, stream)

    _with_scratch((0, B, S, H, Hkv, index), call, dev)
    increment_version(weights)               # written through its address: autograd has to know
    return out


def _distinct_rows(shape, strides, name):
    """A tensor that is written needs unit stride in its last dimension and rows that do not share memory."""
    if strides[-1] != 1 and shape[-1] > 1:
        raise ValueError(f"{name} needs unit stride in the last dimension")
    reach = shape[-1]
    for stride, size in sorted((s, n) for n, s in zip(shape[:-1], strides[:-1]) if n > 1):
        if stride < reach:
            raise ValueError(f"{name} has rows that share memory")
        reach += stride * (size - 1)


def verify_drafts(tokens, target_probs, draft_probs, uniform, parents=None):
    """Which drafted tokens the target model accepts, and one token more, so that tokens come out distributed as the target's.

    tokens (B, n) int64 or int32, 1 <= n <= 64: node 0 is the token sampled last, nodes 1 .. n - 1 are drafts. target_probs
    (B, n, V): the target's distribution behind each node; draft_probs (B, n or n - 1, V), of the same type (float32,
    bfloat16 or float16): the distribution the children of each node were drawn from, None for drafts that were not drawn
    (each counts as certain). uniform (B, n) float32 in [0, 1): entry i decides node i, entry 0 draws the last token. parents
    (n,) or (B, n) int32: the node each follows, an earlier one; None: a chain.

    From node 0 on, the children x of the current node are tried in index order: accepted iff uniform * q(x) * Z < R(x), with R
    the target's distribution and Z = 1 at first; a rejection replaces R by max(R - Z q, 0) and Z by its sum (unless that is
    zero). When none is left the last token is drawn from R: the smallest t with R(0) + .. + R(t) > uniform * sum R. Sums
    and comparisons are in 64 bits.

    Tokens come out distributed as the target's if a node's children were drawn independently of one another; children drawn without
    replacement need other draft probabilities than one row for all of them. Probabilities are finite and not negative: a row that holds
    others gives some token of the vocabulary.

    Returns accepted (B,) int32, the number m of accepted drafts; path (B, n) int32, the nodes from 0 on, then -1; and tokens
    (B, n) int64: the m accepted ones, the drawn one, then -1. Drafts outside the vocabulary are rejected."""
    _forward_only(tokens, target_probs, draft_probs, uniform, parents)
    pn, kind = target_probs.shape, _PROB_TYPES.get(target_probs.dtype)
    if len(pn) != 3 or kind is None or not target_probs.is_cuda:
        raise ValueError("target_probs must be a CUDA float32, bfloat16 or float16 tensor (batch, nodes, vocabulary)")
    B, n, V = pn
    dev = target_probs.device
    if not 1 <= n <= MAX_TOKENS or V == 0:
        raise ValueError(f"expected 1 to {MAX_TOKENS} nodes and a vocabulary, got {n} and {V}")
    wide = tokens.dtype is torch.int64
    if not (wide or tokens.dtype is torch.int32) or tokens.shape != (B, n) or tokens.device != dev:
        raise ValueError(f"tokens must be int64 or int32 ({B}, {n}) on {dev}")
    if uniform.dtype is not torch.float32 or uniform.shape != (B, n) or uniform.device != dev:
        raise ValueError(f"uniform must be float32 ({B}, {n}) on {dev}")
    if draft_probs is not None:
        dn = draft_probs.shape
        if (draft_probs.dtype is not target_probs.dtype or len(dn) != 3 or dn[0] != B or (dn[1] != n and dn[1] != n - 1) or dn[2] != V
                or draft_probs.device != dev):
            raise ValueError(f"draft_probs must be {target_probs.dtype} ({B}, {n - 1} or {n}, {V}) on {dev}")
        if dn[1] == 0:                                       # no drafts
            draft_probs = None
    parents, up, up_stride = _integers(parents, "parents", (B, n), dev, (n,))
    accepted = uniform.new_empty((B,), dtype=torch.int32)
    path = accepted.new_empty((B, n))
    out = tokens.new_empty((B, n)) if wide else uniform.new_empty((B, n), dtype=torch.int64)
    if B == 0:
        return accepted, path, out
    target_probs, uniform = target_probs.resolve_neg(), uniform.resolve_neg()
    if target_probs.stride(2) != 1:
        target_probs = target_probs.contiguous()
    if tokens.stride(1) != 1:
        tokens = tokens.contiguous()
    if uniform.stride(1) != 1:
        uniform = uniform.contiguous()
    ds = None
    if draft_probs is not None:
        draft_probs = draft_probs.resolve_neg()
        if draft_probs.stride(2) != 1:
            draft_probs = draft_probs.contiguous()
        ds = _c_strides(*draft_probs.stride())
    rc = lib.intra_b200_verify_drafts(tokens.data_ptr(), wide, target_probs.data_ptr(), _ptr(draft_probs), kind, uniform.data_ptr(),
                                      up, accepted.data_ptr(), path.data_ptr(), out.data_ptr(), B, n, V,
                                      _c_strides(*target_probs.stride()), ds, tokens.stride(0), uniform.stride(0), up_stride,
                                      dev.index, _raw_stream(dev.index))
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
    all layers, (B, Hkv, S, 128) bfloat16, all of one shape) row lengths[b] + path[b, i] becomes row lengths[b] + i, for every i
    with path[b, i] >= 0. lengths (B,) int32: rows before the tokens' own, as in `tree_attn`; path (B, n) int32, n <= 64, as
    `verify_drafts` returns it. Entries outside 0 .. n - 1 move nothing, and neither does a sequence whose lengths[b] is not in
    0 .. S - n. Other rows stay as they are. The caches must not share memory."""
    caches = [caches] if isinstance(caches, torch.Tensor) else list(caches)
    if not caches:
        return
    _forward_only(lengths, path, *caches)
    first, count = caches[0], len(caches)
    dev, shape, bf16 = first.device, first.shape, torch.bfloat16
    index, alike, pointers = dev.index, first.is_contiguous(), []
    if not first.is_cuda or len(shape) != 4 or shape[3] != 128:
        raise ValueError("INTRA kernels need CUDA bfloat16 tensors (batch, heads, tokens, 128)")
    for x in caches:
        if x.dtype is not bf16:
            raise ValueError("INTRA kernels need CUDA bfloat16 tensors (batch, heads, tokens, 128)")
        if x.shape != shape or x.get_device() != index:
            raise ValueError("caches must agree in shape and device")
        alike = alike and x.is_contiguous()
        pointers.append(x.data_ptr())
    layouts = {x.stride() for x in caches} if not alike else {first.stride()}
    for s in layouts:
        if s[3] != 1 or (s[0] | s[1] | s[2]) & 7:
            raise ValueError("caches need unit stride in the last dimension and 16-byte aligned rows")
        _distinct_rows(shape, s, "a cache")
    order = sorted(pointers)
    if any([p & 15 for p in order]):
        raise ValueError("caches need unit stride in the last dimension and 16-byte aligned rows")
    B, Hkv, S, _ = shape
    if len(path.shape) != 2 or not 1 <= path.shape[1] <= min(MAX_TOKENS, S):
        raise ValueError(f"path must be (batch, n) with n from 1 to {min(MAX_TOKENS, S)}")
    n = path.shape[1]
    path, nodes, path_stride = _integers(path, "path", (B, n), dev)
    lengths, used, _ = _integers(lengths, "lengths", (B,), dev)
    if lengths is None:
        raise ValueError("lengths is needed")
    if B == 0 or Hkv == 0:
        return
    if count > 1:
        span = _byte_span(first)[1] - pointers[0]
        if (len(layouts) > 1 or any([b - a < span for a, b in zip(order, order[1:])])) and _overlapping(caches):
            raise ValueError("caches must not share memory")
    # {batch, token, head}, once for all where they are the same; dimensions of one entry get some positive stride
    strides = [s[d] if shape[d] > 1 else 8 for s in ([first.stride()] if len(layouts) == 1 else [x.stride() for x in caches]) for d in (0, 2, 1)]
    addresses, c_strides = array.array("Q", pointers), array.array("q", strides)
    rc = lib.intra_b200_keep_drafts(addresses.buffer_info()[0], c_strides.buffer_info()[0], 0 if len(layouts) == 1 else 3, count, used,
                                    nodes, path_stride, B, S, Hkv, n, index, _raw_stream(index))
    if rc != 0:
        _raise(rc)
    increment_version(caches)


def evict_cache(k, v, weights, keep, recent=0, lengths=None, out=None):
    """Cuts a cache k, v (B, Hkv, S, 128) down to `keep` rows per head: the last `recent` in use and the heaviest of the others by
    `weights` (B, Hkv, >= S) float32, as `decode_attn_accumulate` leaves them, in their order; ties go to the lower row, NaN counts as
    the heaviest. lengths (B,) int32: rows in use, None: all S (values outside 0 .. S are brought into that range). A sequence with no
    more than `keep` rows keeps them all.

    Returns (k, v, weights, kept): the kept rows, their weights and their old places (B, Hkv, keep) int32. Behind a sequence's
    last row come zeros, and -1 in `kept`; lengths are min(lengths, keep) from then on. `out` = (k, v, weights) writes into the
    caller's tensors of at least `keep` rows, whose rows from `keep` on stay as they are; they must not overlap the inputs."""
    out = None if out is None else tuple(out)
    _forward_only(k, v, weights, lengths, *(out or ()))
    kn, dev, bf16 = k.shape, k.device, torch.bfloat16
    if not k.is_cuda or k.dtype is not bf16 or v.dtype is not bf16 or len(kn) != 4 or kn[3] != 128:
        raise ValueError("INTRA kernels need CUDA bfloat16 tensors (batch, heads, tokens, 128)")
    B, Hkv, S, D = kn
    if v.shape != kn or v.device != dev or S == 0:
        raise ValueError(f"incompatible shapes k={tuple(kn)} v={tuple(v.shape)}")
    wn = weights.shape
    if weights.dtype is not torch.float32 or len(wn) != 3 or wn[0] != B or wn[1] != Hkv or wn[2] < S or weights.device != dev:
        raise ValueError(f"weights must be float32 (batch, KV heads, at least {S}) on {dev}")
    keep, recent = int(keep), int(recent)
    if not 1 <= keep or not 0 <= recent <= keep:
        raise ValueError(f"expected keep >= 1 and recent from 0 to keep, got {keep} and {recent}")
    lengths, used, _ = _integers(lengths, "lengths", (B,), dev)
    k, v = _usable(k), _usable(v)
    weights = weights.resolve_neg()
    if weights.stride(2) != 1:
        weights = weights.contiguous()
    if out is None:
        k2, v2, w2 = k.new_empty((B, Hkv, keep, D)), k.new_empty((B, Hkv, keep, D)), weights.new_empty((B, Hkv, keep))
    else:
        k2, v2, w2 = out
        for x in (k2, v2):
            if x.dtype is not bf16 or x.dim() != 4 or x.shape[:2] != kn[:2] or x.shape[2] < keep or x.shape[3] != D or x.device != dev:
                raise ValueError(f"out needs bfloat16 ({B}, {Hkv}, at least {keep}, 128) for k and v on {dev}")
            if not _rows_usable(x):
                raise ValueError("out needs unit stride in the last dimension and 16-byte aligned rows")
        if w2.dtype is not torch.float32 or w2.dim() != 3 or w2.shape[:2] != kn[:2] or w2.shape[2] < keep or w2.device != dev or w2.is_neg():
            raise ValueError(f"out needs float32 ({B}, {Hkv}, at least {keep}) for the weights on {dev}")
        for x in (k2, v2, w2):
            _distinct_rows(x.shape, x.stride(), "out")
        if _overlapping((k2, v2, w2)) or any(_overlapping((x, y)) for x in (k2, v2, w2) for y in (k, v, weights)):
            raise ValueError("out must not overlap the cache: rows are still read while it is written")
    kept = w2.new_empty((B, Hkv, keep), dtype=torch.int32)
    if B > 0 and Hkv > 0:
        ks, vs, ws = k.stride(), v.stride(), weights.stride()
        rc = lib.intra_b200_evict(k.data_ptr(), v.data_ptr(), weights.data_ptr(), used, k2.data_ptr(), v2.data_ptr(),
                                  w2.data_ptr(), kept.data_ptr(), B, S, Hkv, keep, recent, _c_strides(ks[0], ks[2], ks[1]),
                                  _c_strides(vs[0], vs[2], vs[1]), _c_strides(*ws), _written(k2, (0, 2, 1)), _written(v2, (0, 2, 1)),
                                  _written(w2, (0, 1)), dev.index, _raw_stream(dev.index))
        if rc != 0:
            _raise(rc)
    if out is None:
        return k2, v2, w2, kept
    increment_version((k2, v2, w2))
    return k2[:, :, :keep], v2[:, :, :keep], w2[:, :, :keep], kept


def _written(x, order):
    """Strides of a tensor that is written, those of dimensions of one entry made positive."""
    n, st = x.shape, x.stride()
    s = [st[d] if n[d] > 1 else 8 for d in order]
    return _c_strides(s[0], s[1], s[2] if len(s) > 2 else 0)
