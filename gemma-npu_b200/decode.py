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


def _shape(t, name, shape, dtype, device):
    """A CUDA tensor of this dtype and shape on `device`; returns its data pointer."""
    _need(isinstance(t, torch.Tensor), f"{name} must be a tensor")
    _need(t.dtype == dtype, f"{name} must be {dtype} (got {t.dtype})")
    _need(t.shape == shape, f"{name} must have shape {tuple(shape)} (got {tuple(t.shape)})")
    _need(t.device == device, f"{name} must be on {device} (got {t.device})")
    return t.data_ptr()


def _rows4(t, name, dtype, device):
    """A 4-D tensor of rows with unit stride along the last dimension: (pointer, strides)."""
    _need(isinstance(t, torch.Tensor) and t.dim() == 4, f"{name} must be a 4-D tensor")
    _need(t.dtype == dtype, f"{name} must be {dtype} (got {t.dtype})")
    _need(t.device == device, f"{name} must be on {device} (got {t.device})")
    return t.data_ptr(), _strides4(t, name)


def _strides4(t, name):
    s0, s1, s2, s3 = t.stride()
    n0, n1, n2, n3 = t.shape
    _need(s3 == 1 or n3 <= 1, f"{name} must have unit stride along its last dimension")
    # The stride of a dimension of one element is arbitrary and never used: 0 satisfies every
    # alignment rule.
    return s0 if n0 > 1 else 0, s1 if n1 > 1 else 0, s2 if n2 > 1 else 0


def _cuda(t, name):
    _need(isinstance(t, torch.Tensor) and t.is_cuda, f"{name} must be a CUDA tensor; there is no CPU path")
    return t.device


def _call(device, fn, *args):
    """One C-ABI call on `device`'s current stream, with that device current."""
    if torch.cuda.current_device() == device.index:
        _lib.call(fn, *args, torch.cuda.current_stream(device).cuda_stream)
    else:
        with torch.cuda.device(device):
            _lib.call(fn, *args, torch.cuda.current_stream(device).cuda_stream)


def _workspace(device, nbytes, what):
    _need(nbytes >= 0, what)
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


def _disjoint_rows(t, name, n):
    """The first n dimensions of a tensor that is written must not overlap themselves."""
    for size, stride in zip(t.shape[:n], t.stride()[:n]):
        _need(size <= 1 or stride != 0, f"{name} is written and must not be an expanded view")


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

    Returns out [B, H, N, D] = softmax(scale * q k^T) v, zeros where a token sees nothing.
    With `weights` fp32 [B, KV, S] returns (out, weights_out, draft_weights): weights_out =
    weights plus the probabilities of each committed slot summed over the group's heads and
    the N tokens (in place unless weights_out is given; slots behind lens are left alone),
    draft_weights fp32 [B, KV, N] the same sums of the new tokens."""
    dev = _cuda(q, "q")
    dt = q.dtype
    _need(dt in (torch.bfloat16, torch.float16), f"q must be bfloat16 or float16 (got {dt})")
    qp, qs = _rows4(q, "q", dt, dev)
    kp, ks = _rows4(k, "k", dt, dev)
    vp, vs = _rows4(v, "v", dt, dev)
    knp, kns = _rows4(k_new, "k_new", dt, dev)
    vnp, vns = _rows4(v_new, "v_new", dt, dev)
    B, H, N, D = q.shape
    KV, S = k.shape[1], k.shape[2]
    _need(k.shape == (B, KV, S, D) and v.shape == k.shape, "k and v must be [B, KV, S, D] with q's B and D")
    _need(k_new.shape == (B, KV, N, D) and v_new.shape == k_new.shape, "k_new and v_new must be [B, KV, N, D]")
    _need(KV >= 1 and H % KV == 0, f"H = {H} must be a multiple of KV = {KV}")
    lp = _shape(lens, "lens", (B,), torch.int32, dev)
    _need(lens.is_contiguous(), "lens must be contiguous")
    tp, ts, dp, ds = 0, (0, 0), 0, 0
    if tree is not None:
        _need(isinstance(tree, torch.Tensor) and tree.dim() in (2, 3), "tree must be [N, N] or [B, N, N]")
        tp = _shape(tree, "tree", (N, N) if tree.dim() == 2 else (B, N, N), torch.bool, dev)
        _need(tree.stride(-1) == 1 or N <= 1, "tree must have unit stride along its last dimension")
        ts = (tree.stride(0) if tree.dim() == 3 else 0, tree.stride(-2))
    if depth is not None:
        _need(isinstance(depth, torch.Tensor) and depth.dim() in (1, 2), "depth must be [N] or [B, N]")
        dp = _shape(depth, "depth", (N,) if depth.dim() == 1 else (B, N), torch.int32, dev)
        _need(depth.stride(-1) == 1 or N <= 1, "depth must have unit stride along its last dimension")
        ds = depth.stride(0) if depth.dim() == 2 else 0
    _need(tree is None or window == 0 or depth is not None, "a tree with a window needs the tokens' depths")
    if out is None:
        out = torch.empty((B, H, N, D), dtype=dt, device=dev)
    else:
        _need(out.shape == q.shape, f"out must be {tuple(q.shape)}")
        _disjoint_rows(out, "out", 3)
    op, os_ = _rows4(out, "out", dt, dev)
    wp = wop = dwp = 0
    ws_, wos = (0, 0), (0, 0)
    if weights is not None:
        wp = _shape(weights, "weights", (B, KV, S), torch.float32, dev)
        weights_out = weights if weights_out is None else weights_out
        wop = _shape(weights_out, "weights_out", (B, KV, S), torch.float32, dev)
        _need((weights.stride(2) == 1 and weights_out.stride(2) == 1) or S <= 1,
              "weights and weights_out must have unit stride along S")
        _disjoint_rows(weights_out, "weights_out", 2)
        ws_, wos = weights.stride()[:2], weights_out.stride()[:2]
        if draft_weights is None:
            draft_weights = torch.empty((B, KV, N), dtype=torch.float32, device=dev)
        dwp = _shape(draft_weights, "draft_weights", (B, KV, N), torch.float32, dev)
        _need(draft_weights.is_contiguous(), "draft_weights must be contiguous")
    else:
        _need(weights_out is None and draft_weights is None, "weights_out and draft_weights go with weights")
    if B and N:
        nbytes = _lib.lib().w8_attention_tree_workspace_bytes(B, H, KV, D, S, N, window, weights is not None)
        if nbytes < 0:
            nbytes = 0  # a shape the call itself refuses, with its reason
        ws = _workspace(dev, nbytes, "bad shape")
        args = _lib.ATTENTION_TREE_ARGS.pack(qp, kp, vp, knp, vnp, op, lp, tp, dp, wp, wop, dwp, *qs, *ks, *vs, *kns,
                                             *vns, *os_, *ts, ds, *ws_, *wos, B, H, KV, D, S, N, window, _DTYPES[dt],
                                             scale)
        _call(dev, "w8_attention_tree", args, ws.data_ptr(), nbytes)
    return out if weights is None else (out, weights_out, draft_weights)


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
    dev = _cuda(k, "k")
    dt = k.dtype
    kp, ks = _rows4(k, "k", dt, dev)
    vp, vs = _rows4(v, "v", dt, dev)
    knp, kns = _rows4(k_new, "k_new", dt, dev)
    vnp, vns = _rows4(v_new, "v_new", dt, dev)
    B, KV, S, D = k.shape
    N = k_new.shape[2]
    _need(v.shape == k.shape, "v must have the shape of k")
    _need(k_new.shape == (B, KV, N, D) and v_new.shape == k_new.shape, "k_new and v_new must be [B, KV, N, D]")
    _disjoint_rows(k, "k", 3)
    _disjoint_rows(v, "v", 3)
    lp = _shape(lens, "lens", (B,), torch.int32, dev)
    _need(lens.is_contiguous(), "lens must be contiguous")
    pp, ps, P = 0, 0, N
    if path is not None:
        _need(isinstance(path, torch.Tensor) and path.dim() == 2, "path must be [B, P]")
        P = path.shape[1]
        pp = _shape(path, "path", (B, P), torch.int32, dev)
        _need(path.stride(1) == 1 or P <= 1, "path must have unit stride along P")
        ps = path.stride(0)
        pp = pp if P else lp  # an empty path is a path: nothing is appended, nothing is read
    wp, wst, dwp, dws = 0, (0, 0), 0, (0, 0)
    if weights is not None:
        wp, wst = _shape(weights, "weights", (B, KV, S), torch.float32, dev), weights.stride()[:2]
        _need(weights.stride(2) == 1 or S <= 1, "weights must have unit stride along S")
        _disjoint_rows(weights, "weights", 2)
        if draft_weights is not None:
            dwp = _shape(draft_weights, "draft_weights", (B, KV, N), torch.float32, dev)
            dws = draft_weights.stride()[:2]
            _need(draft_weights.stride(2) == 1 or N <= 1, "draft_weights must have unit stride along N")
    else:
        _need(draft_weights is None, "draft_weights go with weights")
    pop, pos, sp = 0, (0, 0), 0
    if positions is not None:
        _need(seen is not None, "positions go with seen")
        pop, pos = _shape(positions, "positions", (B, KV, S), torch.int32, dev), positions.stride()[:2]
        _need(positions.stride(2) == 1 or S <= 1, "positions must have unit stride along S")
        _disjoint_rows(positions, "positions", 2)
        sp = _shape(seen, "seen", (B,), torch.int32, dev)
        _need(seen.is_contiguous(), "seen must be contiguous")
    if lens_out is None:
        lens_out = torch.empty((B,), dtype=torch.int32, device=dev)
    lop = _shape(lens_out, "lens_out", (B,), torch.int32, dev)
    _need(lens_out.is_contiguous(), "lens_out must be contiguous")
    if B:
        e = k.element_size()
        args = _lib.CACHE_APPEND_ARGS.pack(kp, vp, knp, vnp, lp, pp, wp, dwp, pop, sp, lop, *(s * e for s in ks),
                                           *(s * e for s in vs), *(s * e for s in kns), *(s * e for s in vns), ps, *wst,
                                           *dws, *pos, B, KV, S, N, P, D * e)
        _call(dev, "w8_cache_append", args)
    return lens_out


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
    dev = _cuda(k, "k")
    dt = k.dtype
    kp, ks = _rows4(k, "k", dt, dev)
    vp, vs = _rows4(v, "v", dt, dev)
    B, KV, S, D = k.shape
    _need(v.shape == k.shape, "v must have the shape of k")
    _disjoint_rows(k, "k", 3)
    _disjoint_rows(v, "v", 3)
    lp = _shape(lens, "lens", (B,), torch.int32, dev)
    _need(lens.is_contiguous(), "lens must be contiguous")
    weights_out = torch.empty((B, KV, S), dtype=torch.float32, device=dev) if weights_out is None else weights_out
    positions_out = torch.empty((B, KV, S), dtype=torch.int32, device=dev) if positions_out is None else positions_out
    lens_out = torch.empty((B,), dtype=torch.int32, device=dev) if lens_out is None else lens_out
    ptrs, strides = [], []
    for t, name, d in ((weights, "weights", torch.float32), (positions, "positions", torch.int32),
                       (weights_out, "weights_out", torch.float32), (positions_out, "positions_out", torch.int32)):
        ptrs.append(_shape(t, name, (B, KV, S), d, dev))
        _need(t.stride(2) == 1 or S <= 1, f"{name} must have unit stride along S")
        strides += t.stride()[:2]
    _disjoint_rows(weights_out, "weights_out", 2)
    _disjoint_rows(positions_out, "positions_out", 2)
    lop = _shape(lens_out, "lens_out", (B,), torch.int32, dev)
    _need(lens_out.is_contiguous(), "lens_out must be contiguous")
    if B:
        e = k.element_size()
        nbytes = max(0, _lib.lib().w8_cache_evict_workspace_bytes(B, KV, S, budget))
        ws = _workspace(dev, nbytes, "bad shape")
        args = _lib.CACHE_EVICT_ARGS.pack(kp, vp, ptrs[0], ptrs[1], lp, ptrs[2], ptrs[3], lop, *(s * e for s in ks),
                                          *(s * e for s in vs), *strides, B, KV, S, D * e, budget, sink, recent)
        _call(dev, "w8_cache_evict", args, ws.data_ptr(), nbytes)
    return weights_out, positions_out, lens_out


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
    dev = _cuda(logits, "logits")
    _need(logits.dtype in _DTYPES, f"logits must be float32, bfloat16 or float16 (got {logits.dtype})")
    _need(logits.dim() == 3, "logits must be [B, K, V]")
    B, K, V = logits.shape
    _need(logits.stride(2) == 1 or V <= 1, "logits must have unit stride along V")
    sp = _shape(scores, "scores", (B, K), torch.float32, dev)
    _need(scores.is_contiguous(), "scores must be contiguous")
    fp = None
    if finished is not None:
        fp = _shape(finished, "finished", (B, K), torch.bool, dev)
        _need(finished.is_contiguous(), "finished must be contiguous")
    n = K if n is None else n
    _need(n >= 1, f"n = {n} must be positive")
    _need(order in _ORDERS, f"order must be one of {_ORDERS}")
    out = torch.empty((B, n), dtype=torch.float32, device=dev)
    beam = torch.empty((B, n), dtype=torch.int64, device=dev)
    token = torch.empty((B, n), dtype=torch.int64, device=dev)
    if B:
        nbytes = max(0, _lib.lib().w8_beam_select_workspace_bytes(B, K, V, n))
        ws = _workspace(dev, nbytes, "bad shape")
        _call(dev, "w8_beam_select", logits.data_ptr(), _DTYPES[logits.dtype], logits.stride(0), logits.stride(1), sp,
              fp, pad, cap, B, K, V, n, order == "slot", out.data_ptr(), beam.data_ptr(), token.data_ptr(),
              ws.data_ptr(), nbytes)
    return out, beam, token


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
    first = many[0]
    dev = _cuda(first, "caches")
    _need(isinstance(beam, torch.Tensor) and beam.dim() == 2 and beam.dtype in (torch.int64, torch.int32),
          "beam must be int64 or int32 [B, K]")
    _need(beam.device == dev and beam.is_contiguous(), f"beam must be contiguous on {dev}")
    B, K = beam.shape
    shape, stride, dt = first.shape, first.stride(), first.dtype
    _, strides = _rows4(first, "caches", dt, dev)
    _need(shape[0] == B * K, f"caches must have B * K = {B * K} states (got {shape[0]})")
    _disjoint_rows(first, "caches", 3)
    ptrs = []
    for t in many:
        _need(isinstance(t, torch.Tensor) and t.shape == shape and t.stride() == stride and t.dtype == dt
              and t.device == dev, "caches must share one shape, layout, dtype and device")
        ptrs.append(t.data_ptr())
    _need(len(set(ptrs)) == len(ptrs), "caches must be distinct tensors")
    lp = None
    if lens is not None:
        lp = _shape(lens, "lens", (B * K,), torch.int32, dev)
        _need(lens.is_contiguous(), "lens must be contiguous")
    if B and K and shape[1]:
        e = first.element_size()
        _call(dev, "w8_cache_reorder", (ctypes.c_void_p * len(ptrs))(*ptrs), len(ptrs),
              (ctypes.c_int64 * 3)(*(s * e for s in strides)), beam.data_ptr(), beam.dtype == torch.int64, lp, B, K,
              shape[1], shape[2], shape[3] * e)
    return caches
