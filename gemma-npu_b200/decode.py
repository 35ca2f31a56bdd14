"""Decoding operators: attention over a cache, the cache itself, and beam search.

The prefill side (`kernels.attention_prefill`) attends one prompt to itself.  These attend
new tokens to what came before, and keep it:

    attention_tree(q, k, v, lens, k_new, v_new, ..)  one token, a causal chunk or a drafted
                      tree of tokens over a cache (pipeline.py:133-180 behind cached keys,
                      local_attn.py:44-83), with the accumulated attention weights on request
    cache_append(k, v, k_new, v_new, lens, path)     the accepted path's rows into the cache
    cache_evict(k, v, weights, positions, lens, ..)  cut the cache by accumulated weight
    beam_select(logits, scores, ..)                  beam search's selection over beams and
                      vocabulary, with the final softcap (pipeline.py:335-338) fused
    cache_reorder(caches, beam, lens)                the beams' states follow their parents

A cache is [B, KV, S, D] (unit stride along D, any other strides: head-major, token-major, a
slice of a bigger buffer); `lens` int32 [B] on its device counts each sequence's committed
slots, and what lies behind them is not touched.  q, k_new and v_new have the head-major
layout that `kernels.qkv_norm_rope` returns: for B sequences of N tokens,
`q.unflatten(1, (B, N)).transpose(0, 1)` is the [B, H, N, D] view.

Like every function of `kernels`, these check dtype, shape and layout on the host, run on
torch's current stream of the tensors' device, copy nothing to the host and raise a W8Error
subclass (or ValueError) when a call is refused.  Lengths and indexes are device memory: one
outside its range is skipped and makes `device_status()` raise W8InvalidArgument.  Workspaces
come from torch's allocator per call, so calls on several streams and captured graphs share
nothing.  After one eager call per shape they can be captured into CUDA graphs.
"""
import ctypes

import torch

from . import _lib
from .kernels import _need

_DTYPES = {torch.bfloat16: _lib.W8_BF16, torch.float16: _lib.W8_FP16, torch.float32: _lib.W8_FP32}
_ORDERS = ("score", "slot")

# Checked layouts.  A decode step makes the same few calls over and over, and checking a dozen
# tensors in Python costs more than a short kernel runs: what the checks depend on (shapes,
# strides, dtypes, devices, the plain arguments) is looked up here, and only a layout that was
# never seen is checked in full.  Addresses and values are no part of it: pointers and their
# alignment go to the C ABI with every call.
_CHECKED = {}
_MOST_CHECKED = 4096


def _layout(t):
    return None if t is None else (t.shape, t.stride(), t.dtype, t.device)


def _known(check, key, *args):
    """check(*args) for a layout key, remembered; a key that is None is never remembered."""
    plan = _CHECKED.get(key) if key is not None else None
    if plan is None:
        plan = check(*args)
        if key is not None:
            if len(_CHECKED) >= _MOST_CHECKED:
                _CHECKED.clear()
            _CHECKED[key] = plan
    return plan


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _shape(t, name, shape, dtype, device):
    """A tensor of this dtype and shape on `device`."""
    _need(isinstance(t, torch.Tensor), f"{name} must be a tensor")
    _need(t.dtype == dtype, f"{name} must be {dtype} (got {t.dtype})")
    _need(t.shape == shape, f"{name} must have shape {tuple(shape)} (got {tuple(t.shape)})")
    _need(t.device == device, f"{name} must be on {device} (got {t.device})")


def _vector(t, name, shape, dtype, device):
    _shape(t, name, shape, dtype, device)
    _need(t.is_contiguous(), f"{name} must be contiguous")


def _per_slot(t, name, shape, dtype, device):
    """[batch, kv_heads, n] with unit stride along n: its other strides."""
    _shape(t, name, shape, dtype, device)
    _need(t.stride(2) == 1 or shape[2] <= 1, f"{name} must have unit stride along its last dimension")
    return t.stride()[:2]


def _rows4(t, name, dtype, device):
    """A 4-D tensor of rows with unit stride along the last dimension: its other strides."""
    _need(isinstance(t, torch.Tensor) and t.dim() == 4, f"{name} must be a 4-D tensor")
    _need(t.dtype == dtype, f"{name} must be {dtype} (got {t.dtype})")
    _need(t.device == device, f"{name} must be on {device} (got {t.device})")
    s0, s1, s2, s3 = t.stride()
    n0, n1, n2, n3 = t.shape
    _need(s3 == 1 or n3 <= 1, f"{name} must have unit stride along its last dimension")
    # The stride of a dimension of one element is arbitrary and never used: 0 satisfies every
    # alignment rule.
    return s0 if n0 > 1 else 0, s1 if n1 > 1 else 0, s2 if n2 > 1 else 0


def _cuda(t, name):
    _need(isinstance(t, torch.Tensor) and t.is_cuda, f"{name} must be a CUDA tensor; there is no CPU path")
    return t.device


def _run(device, fn, *args):
    """One C-ABI call on `device`'s current stream, with that device current."""
    index = device.index
    if torch._C._cuda_getDevice() == index:
        status = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(device):
            status = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if status:
        _lib.check(status, fn.__name__)


def _integer(v, name):
    _need(isinstance(v, int), f"{name} must be an integer (got {v!r})")


def _disjoint_rows(t, name, n):
    """The first n dimensions of a tensor that is written must not overlap themselves."""
    for size, stride in zip(t.shape[:n], t.stride()[:n]):
        _need(size <= 1 or stride != 0, f"{name} is written and must not be an expanded view")


def _check_tree(q, k, v, lens, k_new, v_new, tree, depth, window, scale, out, weights, weights_out, draft_weights):
    dev = _cuda(q, "q")
    dt = q.dtype
    _need(dt in (torch.bfloat16, torch.float16), f"q must be bfloat16 or float16 (got {dt})")
    strides = [x for t, name in ((q, "q"), (k, "k"), (v, "v"), (k_new, "k_new"), (v_new, "v_new"))
               for x in _rows4(t, name, dt, dev)]
    B, H, N, D = q.shape
    KV, S = k.shape[1], k.shape[2]
    _need(k.shape == (B, KV, S, D) and v.shape == k.shape, "k and v must be [B, KV, S, D] with q's B and D")
    _need(k_new.shape == (B, KV, N, D) and v_new.shape == k_new.shape, "k_new and v_new must be [B, KV, N, D]")
    _need(KV >= 1 and H % KV == 0, f"H = {H} must be a multiple of KV = {KV}")
    _vector(lens, "lens", (B,), torch.int32, dev)
    ts, ds = (0, 0), 0
    if tree is not None:
        _need(isinstance(tree, torch.Tensor) and tree.dim() in (2, 3), "tree must be [N, N] or [B, N, N]")
        _shape(tree, "tree", (N, N) if tree.dim() == 2 else (B, N, N), torch.bool, dev)
        _need(tree.stride(-1) == 1 or N <= 1, "tree must have unit stride along its last dimension")
        ts = (tree.stride(0) if tree.dim() == 3 else 0, tree.stride(-2))
    if depth is not None:
        _need(isinstance(depth, torch.Tensor) and depth.dim() in (1, 2), "depth must be [N] or [B, N]")
        _shape(depth, "depth", (N,) if depth.dim() == 1 else (B, N), torch.int32, dev)
        _need(depth.stride(-1) == 1 or N <= 1, "depth must have unit stride along its last dimension")
        ds = depth.stride(0) if depth.dim() == 2 else 0
    _integer(window, "window")
    _need(tree is None or window == 0 or depth is not None, "a tree with a window needs the tokens' depths")
    if out is not None:
        _need(out.shape == q.shape, f"out must be {tuple(q.shape)}")
        _disjoint_rows(out, "out", 3)
        strides += _rows4(out, "out", dt, dev)
    else:
        strides += (H * N * D, N * D, D)
    ws, wos = (0, 0), (0, 0)
    if weights is not None:
        ws = _per_slot(weights, "weights", (B, KV, S), torch.float32, dev)
        to = weights if weights_out is None else weights_out
        wos = _per_slot(to, "weights_out", (B, KV, S), torch.float32, dev)
        _disjoint_rows(to, "weights_out", 2)
        if draft_weights is not None:
            _vector(draft_weights, "draft_weights", (B, KV, N), torch.float32, dev)
    else:
        _need(weights_out is None and draft_weights is None, "weights_out and draft_weights go with weights")
    # (a negative size is a shape that the call itself refuses, with its reason)
    nbytes = max(0, _lib.lib().w8_attention_tree_workspace_bytes(B, H, KV, D, S, N, window, weights is not None))
    tail = _lib.ATTENTION_TREE_TAIL.pack(*strides, *ts, ds, *ws, *wos, B, H, KV, D, S, N, window, _DTYPES[dt], scale)
    return dev, (B, H, N, D), (B, KV, N), nbytes, tail, _lib.lib().w8_attention_tree


def attention_tree(q, k, v, lens, k_new, v_new, tree=None, depth=None, window=0, scale=1.0, out=None, weights=None,
                   weights_out=None, draft_weights=None):
    """Attention of N new tokens per sequence over its cache and over one another.

    q bf16 or fp16 [B, H, N, D]; caches k, v [B, KV, S, D] with lens int32 [B] committed slots;
    k_new, v_new [B, KV, N, D] the new tokens' own keys and values, which need not be in the
    cache yet (`cache_append` puts the accepted ones there).  H a multiple of KV; D 64, 128,
    256 or 512; 16-byte aligned, strides multiples of 8.  Token i sees the committed slots and
    - tree=None: the new tokens up to itself (N = 1 is a decode step, N > 1 a causal chunk);
    - tree bool [N, N] or [B, N, N]: the new tokens j with tree[i, j], i.e. its ancestors in
      the drafted tree and itself; a padding draft that no row names may hold anything.
    With window W > 0 a token sees the last W positions only, its own included: slot j stands
    at position j, new token i at lens + depth[i], depth int32 [N] or [B, N] (its number of
    ancestors; needed with a tree, i without one).

    Returns out [B, H, N, D] = softmax(scale * q k^T) v (scale > 0), zeros where a token sees nothing.
    With `weights` fp32 [B, KV, S] returns (out, weights_out, draft_weights): weights_out =
    weights plus the probabilities of each committed slot summed over the group's heads and
    the N tokens (in place unless weights_out is given; slots behind lens are left alone),
    draft_weights fp32 [B, KV, N] the same sums of the new tokens."""
    try:
        key = ("attention_tree", _layout(q), _layout(k), _layout(v), _layout(lens), _layout(k_new), _layout(v_new),
               _layout(tree), _layout(depth), window, scale, _layout(out), _layout(weights), _layout(weights_out),
               _layout(draft_weights))
    except (AttributeError, TypeError):
        key = None
    dev, shape, per_new, nbytes, tail, fn = _known(_check_tree, key, q, k, v, lens, k_new, v_new, tree, depth, window,
                                                   scale, out, weights, weights_out, draft_weights)
    if out is None:
        out = q.new_empty(shape)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    if weights is not None:
        weights_out = weights if weights_out is None else weights_out
        draft_weights = weights.new_empty(per_new) if draft_weights is None else draft_weights
    args = _lib.ATTENTION_TREE_POINTERS.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), k_new.data_ptr(),
                                             v_new.data_ptr(), out.data_ptr(), lens.data_ptr(), _ptr(tree), _ptr(depth),
                                             _ptr(weights), _ptr(weights_out), _ptr(draft_weights)) + tail
    _run(dev, fn, args, _ptr(ws), nbytes)
    return out if weights is None else (out, weights_out, draft_weights)


def _check_append(k, v, k_new, v_new, lens, path, weights, draft_weights, positions, seen, lens_out):
    dev = _cuda(k, "k")
    dt = k.dtype
    e = k.element_size()
    strides = [x * e for t, name in ((k, "k"), (v, "v"), (k_new, "k_new"), (v_new, "v_new"))
               for x in _rows4(t, name, dt, dev)]
    B, KV, S, D = k.shape
    N = k_new.shape[2]
    _need(v.shape == k.shape, "v must have the shape of k")
    _need(k_new.shape == (B, KV, N, D) and v_new.shape == k_new.shape, "k_new and v_new must be [B, KV, N, D]")
    _disjoint_rows(k, "k", 3)
    _disjoint_rows(v, "v", 3)
    _vector(lens, "lens", (B,), torch.int32, dev)
    ps, P = 0, N
    if path is not None:
        _need(isinstance(path, torch.Tensor) and path.dim() == 2, "path must be [B, P]")
        P = path.shape[1]
        _shape(path, "path", (B, P), torch.int32, dev)
        _need(path.stride(1) == 1 or P <= 1, "path must have unit stride along P")
        ps = path.stride(0)
    ws, dws, pos = (0, 0), (0, 0), (0, 0)
    if weights is not None:
        ws = _per_slot(weights, "weights", (B, KV, S), torch.float32, dev)
        _disjoint_rows(weights, "weights", 2)
        if draft_weights is not None:
            dws = _per_slot(draft_weights, "draft_weights", (B, KV, N), torch.float32, dev)
    else:
        _need(draft_weights is None, "draft_weights go with weights")
    if positions is not None:
        _need(seen is not None, "positions go with seen")
        pos = _per_slot(positions, "positions", (B, KV, S), torch.int32, dev)
        _disjoint_rows(positions, "positions", 2)
        _vector(seen, "seen", (B,), torch.int32, dev)
    if lens_out is not None:
        _vector(lens_out, "lens_out", (B,), torch.int32, dev)
    tail = _lib.CACHE_APPEND_TAIL.pack(*strides, ps, *ws, *dws, *pos, B, KV, S, N, P, D * e)
    return dev, B, P, tail, _lib.lib().w8_cache_append


def cache_append(k, v, k_new, v_new, lens, path=None, weights=None, draft_weights=None, positions=None, seen=None,
                 lens_out=None):
    """Put new tokens' rows into the caches, in place, and return the new lengths.

    Rows path[b, 0], path[b, 1], ... of k_new, v_new [B, KV, N, D] go to the slots lens[b],
    lens[b] + 1, ... of k, v [B, KV, S, D] (any dtype whose rows are a multiple of 16 bytes).
    path int32 [B, P] is the accepted path of a drafted tree, ended by a negative entry
    (None: all N tokens in order).  With `weights` fp32 [B, KV, S] the slots take their
    weight from draft_weights [B, KV, N] (None: 0), with `positions` int32 [B, KV, S] the
    positions seen[b], seen[b] + 1, ... (seen int32 [B]: the tokens so far, evicted ones
    included).  Returns lens_out int32 [B] (not `lens` itself)."""
    try:
        key = ("cache_append", _layout(k), _layout(v), _layout(k_new), _layout(v_new), _layout(lens), _layout(path),
               _layout(weights), _layout(draft_weights), _layout(positions), _layout(seen), _layout(lens_out))
    except (AttributeError, TypeError):
        key = None
    dev, B, P, tail, fn = _known(_check_append, key, k, v, k_new, v_new, lens, path, weights, draft_weights, positions,
                                 seen, lens_out)
    if lens_out is None:
        lens_out = lens.new_empty((B,))
    lp = lens.data_ptr()
    # An empty path is a path: nothing is appended and nothing of it is read.
    pp = 0 if path is None else path.data_ptr() if P else lp
    args = _lib.CACHE_APPEND_POINTERS.pack(k.data_ptr(), v.data_ptr(), k_new.data_ptr(), v_new.data_ptr(), lp, pp,
                                           _ptr(weights), _ptr(draft_weights), _ptr(positions),
                                           _ptr(seen) if positions is not None else 0, lens_out.data_ptr()) + tail
    _run(dev, fn, args)
    return lens_out


def _check_evict(k, v, weights, positions, lens, budget, sink, recent, weights_out, positions_out, lens_out):
    dev = _cuda(k, "k")
    dt = k.dtype
    e = k.element_size()
    strides = [x * e for t, name in ((k, "k"), (v, "v")) for x in _rows4(t, name, dt, dev)]
    B, KV, S, D = k.shape
    _need(v.shape == k.shape, "v must have the shape of k")
    _disjoint_rows(k, "k", 3)
    _disjoint_rows(v, "v", 3)
    _vector(lens, "lens", (B,), torch.int32, dev)
    for t, name, d in ((weights, "weights", torch.float32), (positions, "positions", torch.int32),
                       (weights_out, "weights_out", torch.float32), (positions_out, "positions_out", torch.int32)):
        if t is None and name.endswith("out"):
            strides += (KV * S, S)
            continue
        strides += _per_slot(t, name, (B, KV, S), d, dev)
        if name.endswith("out"):
            _disjoint_rows(t, name, 2)
    if lens_out is not None:
        _vector(lens_out, "lens_out", (B,), torch.int32, dev)
    for x, name in ((budget, "budget"), (sink, "sink"), (recent, "recent")):
        _integer(x, name)
    nbytes = max(0, _lib.lib().w8_cache_evict_workspace_bytes(B, KV, S, budget))
    tail = _lib.CACHE_EVICT_TAIL.pack(*strides, B, KV, S, D * e, budget, sink, recent)
    return dev, (B, KV, S), nbytes, tail, _lib.lib().w8_cache_evict


def cache_evict(k, v, weights, positions, lens, budget, sink=0, recent=0, weights_out=None, positions_out=None,
                lens_out=None):
    """Cut the caches of the sequences longer than `budget` to `budget` slots a cache head, by
    accumulated attention weight, in place; returns (weights_out, positions_out, lens_out).

    k, v [B, KV, S, D] (any dtype whose rows are a multiple of 16 bytes); weights fp32 and
    positions int32 [B, KV, S] as `attention_tree` and `cache_append` keep them (positions of
    one head distinct and not negative).  Each head keeps its slots at positions < sink, its
    `recent` last positions, and of the others those with the largest weight (ties to the
    lower slot; NaN counts as -inf); sink + recent <= budget.  The i-th kept slot at or
    behind `budget` moves into the i-th evicted slot below it and nothing else moves: the
    order of a cache's slots means nothing to attention without a window, and positions_out
    says which token stands where.  weights_out and positions_out (new tensors unless given;
    the inputs themselves are allowed) hold 0 and -1 behind the last slot; lens_out =
    min(lens, budget) is not `lens` itself."""
    try:
        key = ("cache_evict", _layout(k), _layout(v), _layout(weights), _layout(positions), _layout(lens), budget, sink,
               recent, _layout(weights_out), _layout(positions_out), _layout(lens_out))
    except (AttributeError, TypeError):
        key = None
    dev, shape, nbytes, tail, fn = _known(_check_evict, key, k, v, weights, positions, lens, budget, sink, recent,
                                          weights_out, positions_out, lens_out)
    weights_out = weights.new_empty(shape) if weights_out is None else weights_out
    positions_out = positions.new_empty(shape) if positions_out is None else positions_out
    lens_out = lens.new_empty(shape[:1]) if lens_out is None else lens_out
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    args = _lib.CACHE_EVICT_POINTERS.pack(k.data_ptr(), v.data_ptr(), weights.data_ptr(), positions.data_ptr(),
                                          lens.data_ptr(), weights_out.data_ptr(), positions_out.data_ptr(),
                                          lens_out.data_ptr()) + tail
    _run(dev, fn, args, ws.data_ptr(), nbytes)
    return weights_out, positions_out, lens_out


def _check_select(logits, scores, finished, pad, n, cap, order):
    dev = _cuda(logits, "logits")
    _need(logits.dtype in _DTYPES, f"logits must be float32, bfloat16 or float16 (got {logits.dtype})")
    _need(logits.dim() == 3, "logits must be [B, K, V]")
    B, K, V = logits.shape
    _need(logits.stride(2) == 1 or V <= 1, "logits must have unit stride along V")
    _vector(scores, "scores", (B, K), torch.float32, dev)
    if finished is not None:
        _vector(finished, "finished", (B, K), torch.bool, dev)
    n = K if n is None else n
    _integer(n, "n")
    _integer(pad, "pad")
    _need(n >= 1, f"n = {n} must be positive")
    _need(order in _ORDERS, f"order must be one of {_ORDERS}")
    nbytes = max(0, _lib.lib().w8_beam_select_workspace_bytes(B, K, V, n))
    mid = (pad, cap, B, K, V, n, order == "slot")
    return dev, (B, n), nbytes, _DTYPES[logits.dtype], logits.stride(0), logits.stride(1), mid, _lib.lib().w8_beam_select


def beam_select(logits, scores, finished=None, pad=0, n=None, cap=0.0, order="score"):
    """Beam search's selection: the n best continuations of each sequence over beams and
    vocabulary, as (scores fp32, beam int64, token int64), each [B, n] (n: the number of beams
    unless given).

    logits fp32, bf16 or fp16 [B, K, V] (unit stride along V), scores fp32 [B, K] the beams'
    log probabilities so far; a continuation's score is scores + log_softmax(y), y = cap *
    tanh(logits / cap) with cap > 0, else the logits; a logit of -inf is an impossible token.
    Best first; equal scores to the lower beam, then the lower token.  A beam with finished
    (bool [B, K]) set has one continuation, the token `pad` at an unchanged score; a beam
    whose score or log sum is not finite has none.  Impossible continuations have score -inf
    and come last.  At most 32 beams and n = 64.

    order="slot" (n = K): the best continuation of a surviving beam stands in that beam's own
    slot, the others fill the free slots, best first: the same continuations, arranged so
    that `cache_reorder` moves as little as can be."""
    try:
        key = ("beam_select", _layout(logits), _layout(scores), _layout(finished), pad, n, cap, order)
    except (AttributeError, TypeError):
        key = None
    dev, shape, nbytes, dt, s0, s1, mid, fn = _known(_check_select, key, logits, scores, finished, pad, n, cap, order)
    out = scores.new_empty(shape)
    beam = torch.empty(shape, dtype=torch.int64, device=dev)
    token = beam.new_empty(shape)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    _run(dev, fn, logits.data_ptr(), dt, s0, s1, scores.data_ptr(), _ptr(finished), *mid, out.data_ptr(),
         beam.data_ptr(), token.data_ptr(), ws.data_ptr(), nbytes)
    return out, beam, token


def _check_reorder(first, beam, lens):
    dev = _cuda(first, "caches")
    _need(isinstance(beam, torch.Tensor) and beam.dim() == 2 and beam.dtype in (torch.int64, torch.int32),
          "beam must be int64 or int32 [B, K]")
    B, K = beam.shape
    _vector(beam, "beam", (B, K), beam.dtype, dev)
    strides = _rows4(first, "caches", first.dtype, dev)
    states, heads, S, D = first.shape
    _need(states == B * K, f"caches must have B * K = {B * K} states (got {states})")
    _disjoint_rows(first, "caches", 3)
    if lens is not None:
        _vector(lens, "lens", (B * K,), torch.int32, dev)
    e = first.element_size()
    return (dev, (ctypes.c_int64 * 3)(*(s * e for s in strides)), beam.dtype == torch.int64,
            (B, K, heads, S, D * e), _lib.lib().w8_cache_reorder)


def cache_reorder(caches, beam, lens=None):
    """Let the states of beam search follow the surviving beams, in place; returns `caches`.

    caches: a tensor or a sequence of distinct tensors [B * K, heads, S, D] of one shape and
    layout (say every layer's K and V; any dtype whose rows are a multiple of 16 bytes); beam
    int64 or int32 [B, K] from `beam_select`.  State i of a sequence takes the first
    lens[parent] slots (lens int32 [B * K] as before the reordering; None: all) of state
    beam[i]; any map is right, swaps and repeated parents included, and a beam that keeps its
    slot costs nothing.  At most 32 beams."""
    many = [caches] if isinstance(caches, torch.Tensor) else list(caches)
    if not many:
        return caches
    try:
        layout = _layout(many[0])
        key = ("cache_reorder", layout, _layout(beam), _layout(lens))
    except (AttributeError, TypeError):
        key = None
    dev, strides, wide, sizes, fn = _known(_check_reorder, key, many[0], beam, lens)
    for t in many:
        _need(isinstance(t, torch.Tensor) and (t is many[0] or _layout(t) == layout),
              "caches must share one shape, layout, dtype and device")
    ptrs = [t.data_ptr() for t in many]
    _need(len(set(ptrs)) == len(ptrs) or not many[0].numel(), "caches must be distinct tensors")
    if sizes[0] and sizes[1] and sizes[2]:
        _run(dev, fn, (ctypes.c_void_p * len(ptrs))(*ptrs), len(ptrs), strides, beam.data_ptr(), wide, _ptr(lens),
             *sizes)
    return caches
