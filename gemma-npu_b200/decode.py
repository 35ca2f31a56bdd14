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
    page_assign(table, lens, free, top, page, ..)    pages of a paged 8-bit cache given out and taken
                      back, on the device
    attention_paged(q, k, v, .., table, lens, k_new, v_new, ..)  attention_tree over such a cache,
                      with a sliding window and sinks
    paged_append(k, v, .., table, lens, k_new, v_new, path)      the accepted path into it
    draft_verify(logits, tokens, uniform, ..)        which drafted tokens stand, and the token after
                      them, from given random numbers

A cache is [B, KV, S, D] (unit stride along D, any other strides: head-major, token-major, a
slice of a bigger buffer); `lens` int32 [B] on its device counts each sequence's committed
slots, and what lies behind them is not touched.  q, k_new and v_new have the head-major
layout that `kernels.qkv_norm_rope` returns: for B sequences of N tokens,
`q.unflatten(1, (B, N)).transpose(0, 1)` is the [B, H, N, D] view.

A paged 8-bit cache (of one layer) is a pool of pages k, v int8 [pages, KV, P, D] with scales
k_scale, v_scale fp32 [pages, KV] (a value is its 8 bits times its page's and head's scale,
which is not negative), P = 16, 32, 64 or 128, and the 16-bit rows of every sequence's last,
partial page, k_tail, v_tail [B, KV, P, D].  table int32 [B, M] names a sequence's pages in
order (negative: none), lens int32 [B] counts its positions: position p is row p % P of page
table[b, p // P], or of the tail where p >= lens // P * P.  Table and lengths are shared by
layers of one kind.

Like every function of `kernels`, these check dtype, shape and layout on the host, run on
torch's current stream of the tensors' device, copy nothing to the host and raise a W8Error
subclass (or ValueError) when a call is refused.  Lengths and indexes are device memory: one
outside its range is skipped and makes `device_status()` raise W8InvalidArgument.  Workspaces
come from torch's allocator per call, so calls on several streams and captured graphs share
nothing.  After one eager call per shape they can be captured into CUDA graphs.

The checks, allocations and packing of arguments are compiled (`_decode.so`, built beside the
library from csrc/decode_binding.cpp): in Python they took 8 to 10 us a call, longer than a
short operator runs.
"""
import importlib.util
import os
import threading

from . import _lib

BINDING_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_decode.so")
_lock = threading.Lock()
_binding = None


def _c():
    """The compiled binding, bound to the loaded library (loaded once per process)."""
    global _binding
    if _binding is None:
        with _lock:
            if _binding is None:
                _lib.lib()
                if not os.path.exists(BINDING_PATH):
                    raise ImportError(f"{BINDING_PATH} is not built; run `python gemma-npu_b200/build.py` "
                                      "(or __graft_entry__.build()) -- there is no CPU fallback")
                import torch  # noqa: F401  (its libraries must be loaded first)

                spec = importlib.util.spec_from_file_location("_decode", BINDING_PATH)
                module = importlib.util.module_from_spec(spec)
                spec.loader.exec_module(module)
                module.bind(_lib.LIB_PATH, _lib.check)
                _binding = module
    return _binding


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
    draft_weights fp32 [B, KV, N] the same sums of the new tokens.  Every row of q counts, a
    padding draft's too.

    A new token's values may be infinite or NaN where some token must not see them, and so may
    slots that no window reaches; the committed slots that one reaches must be finite.  out
    must not overlap the inputs."""
    return (_binding or _c()).attention_tree(q, k, v, lens, k_new, v_new, tree, depth, window, scale, out, weights,
                                             weights_out, draft_weights)


def cache_append(k, v, k_new, v_new, lens, path=None, weights=None, draft_weights=None, positions=None, seen=None,
                 lens_out=None):
    """Put new tokens' rows into the caches, in place, and return the new lengths.

    Rows path[b, 0], path[b, 1], ... of k_new, v_new [B, KV, N, D] go to the slots lens[b],
    lens[b] + 1, ... of k, v [B, KV, S, D] (any dtype whose rows are a multiple of 16 bytes).
    path int32 [B, P] is the accepted path of a drafted tree, ended by a negative entry
    (None: all N tokens in order).  With `weights` fp32 [B, KV, S] the slots take their
    weight from draft_weights [B, KV, N] (None: 0), with `positions` int32 [B, KV, S] the
    positions seen[b], seen[b] + 1, ... (seen int32 [B]: the tokens so far, evicted ones
    included).  Returns lens_out int32 [B] (a tensor apart from lens, seen and path).  k_new and
    v_new must not overlap the caches."""
    return (_binding or _c()).cache_append(k, v, k_new, v_new, lens, path, weights, draft_weights, positions, seen,
                                           lens_out)


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
    min(lens, budget) is a tensor apart from lens."""
    return (_binding or _c()).cache_evict(k, v, weights, positions, lens, budget, sink, recent, weights_out,
                                          positions_out, lens_out)


def beam_select(logits, scores, finished=None, pad=0, n=None, cap=0.0, order="score"):
    """Beam search's selection: the n best continuations of each sequence over beams and
    vocabulary, as (scores fp32, beam int64, token int64), each [B, n] (n: the number of beams
    unless given).

    logits fp32, bf16 or fp16 [B, K, V] (unit stride along V), scores fp32 [B, K] the beams'
    log probabilities so far; a continuation's score is scores + log_softmax(y), y = cap *
    tanh(logits / cap) with cap > 0 (1e-30 to 1e30), else the logits; a logit of -inf is an
    impossible token, under a cap too.
    Best first; equal scores to the lower beam.  Within a beam the order is that of the logits,
    equal ones to the lower token, also where the softcap or the rounding of a score makes the
    scores of different logits equal (far above the cap, say).  A beam with finished
    (bool [B, K]) set has one continuation, the token `pad` at an unchanged score; a beam
    whose score or log sum is not finite has none.  Impossible continuations have score -inf
    and come last.  At most 32 beams and n = 64.

    order="slot" (n = K): the best continuation of a surviving beam stands in that beam's own
    slot, the others fill the free slots, best first: the same continuations, arranged so
    that `cache_reorder` moves as little as can be."""
    return (_binding or _c()).beam_select(logits, scores, finished, pad, n, cap, order)


def cache_reorder(caches, beam, lens=None):
    """Let the states of beam search follow the surviving beams, in place; returns `caches`.

    caches: a tensor or a sequence of distinct tensors [B * K, heads, S, D] of one shape and
    layout (say every layer's K and V; any dtype whose rows are a multiple of 16 bytes); beam
    int64 or int32 [B, K] from `beam_select`.  State i of a sequence takes the first
    lens[parent] slots (lens int32 [B * K] as before the reordering; None: all) of state
    beam[i]; any map is right, swaps and repeated parents included, and a beam that keeps its
    slot costs nothing.  At most 32 beams."""
    (_binding or _c()).cache_reorder(caches if isinstance(caches, (list, tuple)) else [caches], beam, lens)
    return caches


def page_assign(table, lens, free, top, page, room=1, active=None, window=0, sink=0):
    """Give every request the pages that its next `room` tokens need, take back those that it
    does not need, all on the device; returns ok bool [B].

    table int32 [B, M] and the stack of free pages, free int32 [F] with top int32 [1] (free[0] to
    free[top - 1] are free), are updated in place.  A request needs the pages (of `page` tokens:
    16, 32, 64 or 128) of its first lens[b] + room positions; none if active (bool [B]) says that
    it has ended; and with window W > 0 not those that lie wholly before the window of position
    lens[b] and behind the first `sink` positions.  What a request holds and does not need goes
    back first, then what is missing is given out, both in the order of the requests and their
    tables, the stack's top first.  ok[b]: the request has all that it needs.  It is served if what
    it and all requests before it miss is there, and always if it misses nothing; one that needs
    more than M pages is not served.  A page belongs to one request; at most 8192 requests."""
    return (_binding or _c()).page_assign(table, lens, free, top, page, room, active, window, sink)


def attention_paged(q, k, v, k_scale, v_scale, k_tail, v_tail, table, lens, k_new, v_new, tree=None, depth=None,
                    window=0, sink=0, scale=1.0, out=None):
    """`attention_tree` over a paged 8-bit cache: N new tokens per sequence over its committed
    positions and over one another; returns out [B, H, N, D].

    q, k_new, v_new, tree, depth, scale and out as for attention_tree (bf16 or fp16, the tails
    alike; D 64, 128, 256 or 512; 16-byte aligned, strides multiples of 8, pages' of 16).  With
    window W > 0 a token sees the last W positions, its own included, and the positions below
    `sink`, which stay visible (a tree then needs its depths).  Pages that no token sees are not
    read and need not be in the table; a page that is needed and missing is skipped and
    reported by `device_status`.

    k_new and v_new may be infinite or NaN where some token must not see them; tail rows that a
    window reaches, or sinks, must be finite.  Only q and out may be expanded or have other than
    positive strides.  out must not overlap the inputs.  Inference only."""
    return (_binding or _c()).attention_paged(q, k, v, k_scale, v_scale, k_tail, v_tail, table, lens, k_new, v_new,
                                              tree, depth, window, sink, scale, out)


def paged_append(k, v, k_scale, v_scale, k_tail, v_tail, table, lens, k_new, v_new, path=None, count=None,
                 lens_out=None):
    """Put new tokens' rows into a paged 8-bit cache, in place, and return the new lengths.

    Rows path[b, 0], path[b, 1], ... of k_new, v_new [B, KV, N, D] (bf16 or fp16) go to the
    positions lens[b], lens[b] + 1, ...; path int32 [B, steps] ends at a negative entry (None: all
    N tokens in order), and with count int32 [B] at count[b] entries (prompts of several lengths).
    They wait in the tail as they are; a page that becomes full is rounded to 8 bits at once, per
    head: scale = m / 127 for its largest magnitude m, values round(127 x / m), halves to even.  A
    page with an infinity or a NaN gets a scale of NaN.  The page must be in the table
    (`page_assign`), and there only once: one that is not is lost and reported by `device_status`.  A
    path's entry of N or more puts a row of zeros, which counts, and is reported too.
    Returns lens_out int32 [B] (a tensor apart from lens, path, count and table).  k_new and v_new must not overlap the
    cache."""
    return (_binding or _c()).paged_append(k, v, k_scale, v_scale, k_tail, v_tail, table, lens, k_new, v_new, path,
                                           count, lens_out)


def draft_verify(logits, tokens, uniform, parent=None, draft=None, temperature=1.0, cap=0.0):
    """Which nodes of a drafted tree stand, and the token after them: (path int32 [B, N], taken
    int32 [B], token int64 [B]).

    logits fp32, bf16 or fp16 [B, N, V] (unit stride along V) are the target's after each node,
    tokens int64 [B, N] the nodes' tokens (node 0's is committed already), parent int32 [N] or
    [B, N] each node's parent, which comes before it (negative: the node is not there; None: a
    chain).  Speculative sampling: with p = softmax(y / temperature), y = cap * tanh(logits /
    cap) with cap > 0 (1e-3 to 1e6), else the logits, and q = softmax(draft / temperature) of the
    draft model's logits [B, N, V] after the same node, a node's children c in order:
    c stands if uniform[b, c] * q(its token) < w(its token), w = p at first, and if not w becomes
    max(w - q, 0) over its sum.  draft=None: the drafts were chosen, not sampled, q is 1 at the
    child's token.  From the last node that stands the token is drawn from w, the first whose
    running sum exceeds uniform[b, 0] of the whole.  uniform fp32 [B, N] in [0, 1).  All this in 64
    bits: w stays as it is where rejections would leave less than 1e-13 of p, and weights below
    2^-1000 of a row's largest count as 0.

    The tokens then have the target's distribution: without `draft` whatever the drafts, with it if
    a node's children are independent draws from its q (the same token may be drawn twice).  The
    draft model's likeliest tokens, or draws without replacement, are chosen drafts.

    temperature=0 (else 1e-3 to 1e3): a child stands if it is the largest logit (equal ones: the
    lowest token), which is also the token after the last; uniform may be None.  A logit of -inf
    is an impossible token.  A node whose target logits hold a NaN or no finite largest one ends
    the walk with token -1; one whose draft logits do keeps no child.  path (node 0 first, then
    -1) is what `cache_append` and `paged_append` take.  At most 1024 nodes; a token outside [0, V)
    does not stand and is reported by `device_status`."""
    return (_binding or _c()).draft_verify(logits, tokens, uniform, parent, draft, temperature, cap)
