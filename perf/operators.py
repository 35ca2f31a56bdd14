"""What the decoding operators are timed on: attention of one token, a chunk or a tree of
drafted tokens over a cache, appending to the cache, evicting from it by accumulated
attention weight, beam search's selection and the reordering of its states.

`run` computes an operator in plain torch operations where `own` is false and makes the
framework's own call where it is true; `exact` is the same in 64 bits, written apart.
"""
import importlib
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_w8 = None


def _kernels():
    global _w8
    if _w8 is None:
        _w8 = importlib.import_module("gemma-npu_b200")
    return _w8


# ---------------------------------------------------------------- cases
# H, KV, D: query heads, cache heads, head size; S: slots of the cache, N: new tokens of each
# sequence; `spread`: the sequences' lengths run from S down to (1 - spread) S; `room`: slots
# behind the longest sequence; `empty`: sequences with nothing in the cache; `pad`: drafts of
# each tree that stand for nothing (their K / V rows hold whatever was in memory).
def listed():
    return [
        # One user, one token: a full-attention layer (head size 512, one cache head) behind a
        # prompt of 3658 tokens; the call's latency counts.
        dict(name="attend one token", op="attention", B=1, H=8, KV=1, D=512, S=3658, room=438, spread=0.0, empty=0,
             N=1, tree=False, pad=0, window=0, dtype="bf16", weights=False),
        # A serving batch's decode step with ragged lengths, the attention weights accumulated
        # for eviction: bound by reading the cache.
        dict(name="attend batch, weights", op="attention", B=32, H=32, KV=8, D=128, S=8191, room=1, spread=0.75,
             empty=0, N=1, tree=False, pad=0, window=0, dtype="bf16", weights=True),
        # Verifying trees of 60 drafts for 16 sequences: 480 query rows share each cache head.
        dict(name="attend tree of 60", op="attention", B=16, H=16, KV=2, D=256, S=4000, room=96, spread=0.5, empty=1,
             N=64, tree=True, pad=4, window=0, dtype="bf16", weights=False),
        # A 512-row micro-batch of a prompt behind the 3146 tokens before it, on a sliding layer.
        dict(name="attend chunk, sliding", op="attention", B=1, H=8, KV=1, D=256, S=3146, room=512, spread=0.0,
             empty=0, N=512, tree=False, pad=0, window=512, dtype="bf16", weights=False),
        # One token of every sequence of a small batch goes into the cache.
        dict(name="append one token", op="append", B=8, KV=1, D=256, S=4096, N=1, P=1, spread=0.5, dtype="bf16",
             weights=False),
        # The accepted paths of drafted trees of a serving batch, with weights and positions.
        dict(name="append paths", op="append", B=256, KV=8, D=128, S=1021, N=64, P=17, spread=0.5, dtype="bf16",
             weights=True),
        # One prompt's cache head cut from 3658 slots to 1024.
        dict(name="evict one prompt", op="evict", B=1, KV=1, D=256, S=3658, budget=1024, sink=4, recent=128,
             spread=0.0, dtype="bf16"),
        # A serving batch cut to 4096 slots a cache head, some sequences already short enough.
        dict(name="evict batch", op="evict", B=24, KV=8, D=128, S=16001, budget=4096, sink=4, recent=512, spread=0.9,
             dtype="bf16"),
        # Four beams of one user over the 262144-wide head's logits.
        dict(name="select 4 beams", op="select", B=1, K=4, V=262144, n=4, dtype="fp32", cap=0.0, finished=False,
             first=False, order="score"),
        # 24 users with eight beams each, bf16 logits of the int8 head with the softcap, twice
        # as many continuations as beams (so that ended ones can be set aside).
        dict(name="select 24 x 8 beams", op="select", B=24, K=8, V=262144, n=16, dtype="bf16", cap=30.0,
             finished=True, first=False, order="score"),
        # Four beams of one user: the caches of a few layers follow the surviving beams.
        dict(name="reorder 4 beams", op="reorder", B=1, K=4, KV=1, D=256, S=2048, layers=4, moved=2, spread=0.3,
             dtype="bf16"),
        # 16 users with eight beams, the K and V of sixteen layers.
        dict(name="reorder 16 x 8 beams", op="reorder", B=16, K=8, KV=2, D=128, S=1000, layers=16, moved=3,
             spread=0.3, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "append", "evict", "evict", "select", "select", "reorder"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "attention":
        D = rng.choice([64, 128, 256, 512])
        KV = rng.choice([1, 1, 2, 4, 8])
        G = rng.choice([1, 2, 3, 4, 5, 8])
        kind = rng.choice(["token", "token", "chain", "tree", "tree"])
        N = 1 if kind == "token" else _log(rng, 2, 128)
        B = _log(rng, 1, 48)
        # at most 64 MB of keys of one call, and 2^26 scores
        most = min(16384, (1 << 25) // (B * KV * D), (1 << 26) // (B * KV * G * N))
        S = _log(rng, 1, max(2, most))
        empty = rng.choice([0, 0, 1]) if B > 1 else 0
        return dict(op=op, B=B, H=KV * G, KV=KV, D=D, S=S, room=rng.randint(0, 200), spread=rng.choice([0.0, 0.5, 0.95]),
                    empty=empty, N=N, tree=kind == "tree", pad=rng.randint(0, N // 4) if kind == "tree" else 0,
                    window=rng.choice([0, 0, 64, 300, 512]), dtype=dtype, weights=rng.random() < 0.35)
    if op == "append":
        N = _log(rng, 1, 64)
        return dict(op=op, B=_log(rng, 1, 256), KV=rng.choice([1, 2, 5, 8]), D=rng.choice([64, 128, 256, 512]),
                    S=_log(rng, 80, 1000), N=N, P=rng.randint(1, N), spread=0.5, dtype=dtype,
                    weights=rng.random() < 0.5)
    if op == "evict":
        S = _log(rng, 2, 16384)
        budget = rng.randint(1, S)
        recent = rng.randint(0, budget)
        KV, D = rng.choice([1, 2, 8]), rng.choice([64, 128, 256])
        B = min(_log(rng, 1, 24), (1 << 28) // (KV * D * S))
        return dict(op=op, B=B, KV=KV, D=D, S=S, budget=budget,
                    sink=rng.randint(0, min(8, budget - recent)), recent=recent, spread=rng.choice([0.0, 0.9]), dtype=dtype)
    if op == "select":
        K = rng.choice([1, 2, 3, 4, 5, 8, 16])
        V = _log(rng, 64, 262144)
        first = rng.random() < 0.2
        order = rng.choice(["score", "slot"])
        return dict(op=op, B=_log(rng, 1, 24), K=K, V=V, n=K if order == "slot" else rng.choice([K, 2 * K]),
                    dtype=rng.choice(["fp32", "bf16", "fp16"]), cap=rng.choice([0.0, 30.0]),
                    finished=rng.random() < 0.4 and not first, first=first, order=order)
    K, KV, D = rng.choice([2, 3, 4, 8]), rng.choice([1, 2, 4]), rng.choice([64, 128, 256])
    S, layers = _log(rng, 1, 1024), rng.randint(1, 12)
    B = min(_log(rng, 1, 16), (1 << 29) // (K * KV * D * S * layers) + 1)
    return dict(op=op, B=B, K=K, KV=KV, D=D, S=S, layers=layers, moved=rng.randint(1, K - 1), spread=0.3, dtype=dtype)


# ---------------------------------------------------------------- states
def _lens(c):
    """The sequences' lengths of a case, longest first (a seed shuffles them)."""
    B, S = c["B"], c["S"]
    lens = [max(1, int(round(S * (1.0 - c["spread"] * b / max(1, B - 1))))) for b in range(B)]
    for b in range(c.get("empty", 0)):
        lens[B - 1 - b] = 0
    return lens


def _rows(gen, shape, dtype, scale=1.0):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).mul_(scale).to(dtype)


def _trees(rng, B, N, pad):
    """Ancestor masks and depths of B random trees of N - pad drafts, parents before children."""
    mask, depth = np.zeros((B, N, N), dtype=bool), np.zeros((B, N), dtype=np.int32)
    for b in range(B):
        for i in range(N - pad):
            parent = int(rng.integers(max(-1, i - 8), i)) if i else -1
            if parent >= 0:
                mask[b, i] = mask[b, parent]
                depth[b, i] = depth[b, parent] + 1
            mask[b, i, i] = True
    return mask, depth


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    dt = DTYPES[c["dtype"]]
    s = {"case": c}
    op = c["op"]

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    if op == "select":
        B, K, V = c["B"], c["K"], c["V"]
        s["logits"] = _rows(gen, (B, K, V), dt, 4.0)
        s["scores"] = torch.sort(torch.randn((B, K), generator=gen, device="cuda") * 3 - 20, descending=True)[0]
        if c["first"]:  # the first step: every beam but one is impossible
            s["scores"][:, 1:] = -math.inf
        s["finished"] = None
        if c["finished"]:
            s["finished"] = torch.rand((B, K), generator=gen, device="cuda") < 0.2
        return s
    if op == "reorder":
        B, K = c["B"], c["K"]
        shape = (B * K, c["KV"], c["S"], c["D"])
        s["caches"] = [_rows(gen, shape, dt) for _ in range(2 * c["layers"])]
        # Survivors keep their slots; each of the `moved` other slots takes some survivor's state.
        order = np.argsort(rng.random((B, K)), axis=1)
        beam = np.tile(np.arange(K), (B, 1))
        keep = K - c["moved"]
        src = np.take_along_axis(order, rng.integers(0, keep, (B, c["moved"])), axis=1)
        np.put_along_axis(beam, order[:, keep:], src, axis=1)
        s["beam"] = torch.from_numpy(beam).cuda()
        s["lens"] = ints(np.repeat(rng.permutation(_lens(c)), K))
        return s

    B, KV, D, S = c["B"], c["KV"], c["D"], c["S"]
    lens = rng.permutation(_lens(c))
    s["lens"] = ints(lens)
    if op == "attention":
        H, N, cap = c["H"], c["N"], S + c["room"]
        # Keys of unit mean square per element and queries that give scores of a deviation of 2.
        s["k"], s["v"] = _rows(gen, (B, KV, cap, D), dt), _rows(gen, (B, KV, cap, D), dt)
        behind = torch.arange(cap, device="cuda")[None, :] >= s["lens"][:, None]
        for name in ("k", "v"):  # what was in memory behind each sequence
            s[name].masked_fill_(behind[:, None, :, None], math.nan)
        s["q"] = _rows(gen, (B, H, N, D), dt, 2.0)
        s["k_new"], s["v_new"] = _rows(gen, (B, KV, N, D), dt), _rows(gen, (B, KV, N, D), dt)
        s["scale"] = D ** -0.5
        s["tree"] = s["depth"] = None
        if c["tree"]:
            mask, depth = _trees(rng, B, N, c["pad"])
            s["tree"], s["depth"] = torch.from_numpy(mask).cuda(), torch.from_numpy(depth).cuda()
            if c["pad"]:
                for name in ("k_new", "v_new"):
                    s[name][:, :, N - c["pad"]:] = math.nan
        s["weights"] = s["weights_out"] = None
        if c["weights"]:
            s["weights"] = torch.rand((B, KV, cap), generator=gen, device="cuda")
            s["weights_out"] = torch.zeros((B, KV, cap), device="cuda")
        return s
    if op == "append":
        N, P, cap = c["N"], c["P"], S + c["N"]
        s["k"], s["v"] = _rows(gen, (B, KV, cap, D), dt), _rows(gen, (B, KV, cap, D), dt)
        s["k_new"], s["v_new"] = _rows(gen, (B, KV, N, D), dt), _rows(gen, (B, KV, N, D), dt)
        path = np.sort(np.argsort(rng.random((B, N)), axis=1)[:, :P], axis=1)
        taken = np.arange(P)[None, :] <= (np.arange(B) % P)[rng.permutation(B)][:, None]
        s["path"] = None if N == 1 else ints(np.where(taken, path, -1))
        s["weights"] = s["draft_weights"] = s["positions"] = s["seen"] = None
        if c["weights"]:
            s["weights"] = torch.rand((B, KV, cap), generator=gen, device="cuda")
            s["draft_weights"] = torch.rand((B, KV, N), generator=gen, device="cuda")
            s["positions"] = torch.arange(cap, device="cuda", dtype=torch.int32).repeat(B, KV, 1)
            s["seen"] = s["lens"] + 100
        return s
    # Heavy-tailed weights with some never-attended slots; the slots' positions in the order an
    # earlier eviction left them in.
    s["k"], s["v"] = _rows(gen, (B, KV, S, D), dt), _rows(gen, (B, KV, S, D), dt)
    w = torch.exp(3 * torch.randn((B, KV, S), generator=gen, device="cuda"))
    s["weights"] = w.masked_fill_(torch.rand((B, KV, S), generator=gen, device="cuda") < 0.02, 0.0)
    at = torch.arange(S, device="cuda", dtype=torch.int32) * 2
    swap = torch.argsort(torch.rand((B, KV, S // 2), generator=gen, device="cuda"), dim=-1)
    s["positions"] = at.repeat(B, KV, 1)
    s["positions"][:, :, :S // 2] = at[swap]
    s["weights_out"] = torch.empty_like(s["weights"])
    s["positions_out"] = torch.empty_like(s["positions"])
    return s


# ---------------------------------------------------------------- one pass
def _attention(c, s):
    B, H, N, D = s["q"].shape
    KV, cap = s["k"].shape[1], s["k"].shape[2]
    G, dev = H // KV, s["q"].device
    q = s["q"].float().reshape(B, KV, G * N, D)
    slot = torch.arange(cap, device=dev)
    lens = s["lens"].long()[:, None, None]
    i = torch.arange(N, device=dev)
    depth = i[None, :].expand(B, N) if s["depth"] is None else s["depth"].long()
    seen = slot[None, None, :] < lens                                           # [B, 1, cap]
    tree = (i[None, :] <= i[:, None]).expand(B, N, N) if s["tree"] is None else s["tree"]
    old = seen.expand(B, N, cap)
    if c["window"]:
        old = old & (slot[None, None, :] > lens + depth[:, :, None] - c["window"])
        tree = tree & (depth[:, None, :] > depth[:, :, None] - c["window"])
    see = torch.cat([old, tree], 2)[:, None, None].expand(B, KV, G, N, cap + N).reshape(B, KV, G * N, cap + N)
    used = torch.cat([seen[:, 0], tree.any(1)], 1)[:, None, :, None]            # keys that some row may see
    k = torch.cat([s["k"].float(), s["k_new"].float()], 2)
    v = torch.where(used, torch.cat([s["v"].float(), s["v_new"].float()], 2), 0.0)
    x = (q @ k.transpose(2, 3) * s["scale"]).masked_fill(~see, -math.inf)
    top = x.amax(3, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(3, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    o = (p @ v).reshape(B, H, N, D).to(s["q"].dtype)
    if s["weights"] is None:
        return o
    w = p.sum(2)
    out = torch.where(seen, s["weights"] + w[:, :, :cap], s["weights_out"])
    return o, out, w[:, :, cap:]


def _append(c, s):
    B, KV, cap, D = s["k"].shape
    N = s["k_new"].shape[2]
    dev = s["k"].device
    path = torch.arange(N, device=dev)[None].expand(B, N) if s["path"] is None else s["path"].long()
    P = path.shape[1]
    ok = (path >= 0).long().cumprod(1).bool()
    j = torch.arange(P, device=dev)
    slot = (s["lens"].long()[:, None] + j)[:, None].expand(B, KV, P)            # room for P slots is there
    draft = path.clamp(min=0)[:, None].expand(B, KV, P)
    ok3 = ok[:, None].expand(B, KV, P)
    for a, b in (("k", "k_new"), ("v", "v_new")):                               # what is not taken writes what is there
        at = slot[..., None].expand(B, KV, P, D)
        rows = s[b].gather(2, draft[..., None].expand(B, KV, P, D))
        s[a].scatter_(2, at, torch.where(ok3[..., None], rows, s[a].gather(2, at)))
    lens = s["lens"] + ok.sum(1, dtype=torch.int32)
    if s["weights"] is None:
        return s["k"], s["v"], lens
    w = torch.where(ok3, s["draft_weights"].gather(2, draft), s["weights"].gather(2, slot))
    s["weights"].scatter_(2, slot, w)
    at = (s["seen"].long()[:, None] + j).int()[:, None].expand(B, KV, P)
    s["positions"].scatter_(2, slot, torch.where(ok3, at, s["positions"].gather(2, slot)))
    return s["k"], s["v"], lens, s["weights"], s["positions"]


def _evict(c, s):
    w, pos, budget = s["weights"], s["positions"], c["budget"]
    B, KV, S = w.shape
    dev = w.device
    slot = torch.arange(S, device=dev)
    lens = s["lens"].long()[:, None, None]
    valid = (slot < lens).expand(B, KV, S)
    last = torch.where(valid, pos, -1).amax(2, keepdim=True)
    kind = valid.int() + (valid & ((pos < c["sink"]) | (pos > last - c["recent"]))).int()
    key = torch.where(valid & ~w.isnan(), w, -math.inf)
    order = torch.argsort(key, dim=2, descending=True, stable=True)
    order = order.gather(2, torch.argsort(kind.gather(2, order), dim=2, descending=True, stable=True))
    keep = torch.zeros((B, KV, S), dtype=torch.bool, device=dev).scatter_(2, order[:, :, :budget], True) & valid
    cut = valid.any(2, keepdim=True) & (lens > budget)
    hole = cut & ~keep & (slot < budget)
    mover = cut & keep & (slot >= budget)
    movers = torch.argsort(mover.int(), dim=2, descending=True, stable=True)
    src = torch.where(hole, movers.gather(2, (hole.long().cumsum(2) - 1).clamp(min=0)), slot)[:, :, :budget]
    for name in ("k", "v"):
        x = s[name]
        x[:, :, :budget] = x.gather(2, src[..., None].expand(*src.shape, x.shape[3]))
    left = (slot[:budget] < lens)
    s["weights_out"].fill_(0.0)[:, :, :budget] = torch.where(left, w.gather(2, src), 0.0)
    s["positions_out"].fill_(-1)[:, :, :budget] = torch.where(left, pos.gather(2, src), -1)
    return s["k"], s["v"], s["weights_out"], s["positions_out"], s["lens"].clamp(max=budget)


def _select(c, s):
    x = s["logits"]
    B, K, V = x.shape
    n, dev = c["n"], x.device
    token = torch.arange(V, device=dev)
    cum = s["scores"].double()[:, :, None]
    capped = (lambda t: c["cap"] * torch.tanh(t / c["cap"])) if c["cap"] else (lambda t: t)
    y = capped(x.double())
    top = y.amax(2, keepdim=True)
    z = top + torch.log(torch.exp(y - top).sum(2, keepdim=True))
    del y
    # Within a beam the order is that of the logits, ties to the lower token.
    bits = x.float().view(torch.int32).long()
    key = torch.where(x == 0, 0x80000000, torch.where(bits < 0, ~bits & 0xFFFFFFFF, bits + 0x80000000))
    key = torch.where(torch.isfinite(z) & torch.isfinite(cum), key, 0)
    if s["finished"] is not None:
        key = torch.where(s["finished"][:, :, None], (token == 0).long(), key)
    m = min(n, V)
    best = torch.topk(key * (1 << 31) + (0x7FFFFFFF - token), m, dim=2)[0]
    pick = 0x7FFFFFFF - (best & 0x7FFFFFFF)
    total = cum + capped(x.gather(2, pick).double()) - z
    if s["finished"] is not None:
        total = torch.where(s["finished"][:, :, None], torch.where(pick == 0, cum, -math.inf), total)
    total = torch.where(torch.isfinite(total), total, -math.inf)
    flat = (pick + torch.arange(K, device=dev)[None, :, None] * V).reshape(B, -1)
    flat, at = torch.sort(flat, dim=1)
    total = total.reshape(B, -1).gather(1, at)
    total, at = torch.sort(total, dim=1, descending=True, stable=True)
    total, flat = total[:, :n], flat.gather(1, at[:, :n])
    beam, token = flat // V, flat % V
    if c["order"] == "slot":
        same = beam[:, :, None] == beam[:, None, :]
        again = torch.tril(same, -1).any(2)                                     # a better one has this parent too
        free = ~(beam[:, :, None] == torch.arange(K, device=dev)).any(1)
        frees = torch.argsort(free.int(), dim=1, descending=True, stable=True)
        slot = torch.where(again, frees.gather(1, (again.long().cumsum(1) - 1).clamp(min=0)), beam)
        back = torch.argsort(slot, dim=1)
        total, beam, token = total.gather(1, back), beam.gather(1, back), token.gather(1, back)
    return total.float(), beam, token


def _reorder(c, s):
    K, S = c["K"], c["S"]
    rows = torch.arange(s["beam"].numel(), device=s["beam"].device)
    src = (s["beam"] + rows.reshape(-1, K)[:, :1]).reshape(-1)
    copied = (torch.arange(S, device=src.device) < s["lens"][src][:, None])[:, None, :, None]
    for x in s["caches"]:
        x.copy_(torch.where(copied, x[src], x))
    return s["caches"]


PLAIN = {"attention": _attention, "append": _append, "evict": _evict, "select": _select, "reorder": _reorder}


def run(state):
    s, c = state, state["case"]
    if not own:
        return PLAIN[c["op"]](c, s)
    w8 = _kernels()
    op = c["op"]
    if op == "attention":
        return w8.attention_tree(s["q"], s["k"], s["v"], s["lens"], s["k_new"], s["v_new"], tree=s["tree"],
                                 depth=s["depth"], window=c["window"], scale=s["scale"], weights=s["weights"],
                                 weights_out=s["weights_out"])
    if op == "append":
        lens = w8.cache_append(s["k"], s["v"], s["k_new"], s["v_new"], s["lens"], path=s["path"],
                               weights=s["weights"], draft_weights=s["draft_weights"], positions=s["positions"],
                               seen=s["seen"])
        return (s["k"], s["v"], lens) + ((s["weights"], s["positions"]) if s["weights"] is not None else ())
    if op == "evict":
        w, pos, lens = w8.cache_evict(s["k"], s["v"], s["weights"], s["positions"], s["lens"], c["budget"],
                                      sink=c["sink"], recent=c["recent"], weights_out=s["weights_out"],
                                      positions_out=s["positions_out"])
        return s["k"], s["v"], w, pos, lens
    if op == "select":
        return w8.beam_select(s["logits"], s["scores"], finished=s["finished"], n=c["n"], cap=c["cap"],
                              order=c["order"])
    return w8.cache_reorder(s["caches"], s["beam"], lens=s["lens"])


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    c = case
    op = c["op"]
    size = 4 if c["dtype"] == "fp32" else 2
    if op == "select":
        rows = c["B"] * c["K"]
        return {"bytes": rows * c["V"] * size + rows * 5 + c["B"] * c["n"] * 20, "flops": 4.0 * rows * c["V"]}
    lens = _lens(c)
    row = c["D"] * size
    if op == "attention":
        N, W, G = c["N"], c["window"], c["H"] // c["KV"]
        keys = sum(min(n, W + N - 2) if W else n for n in lens)
        pairs = sum((min(n, W - 1) if W else n) * N for n in lens) + c["B"] * N * (1 if N == 1 else N / 2)
        by = c["KV"] * 2 * row * (keys + c["B"] * N) + 2 * c["B"] * c["H"] * N * row + 4 * c["B"]
        by += c["B"] * N * N if c["tree"] else 0
        by += 4 * c["KV"] * (2 * keys + c["B"] * N) if c["weights"] else 0
        return {"bytes": by, "flops": 4.0 * c["KV"] * G * c["D"] * pairs}
    if op == "append":
        rows = sum(b % c["P"] + 1 for b in range(c["B"]))
        return {"bytes": 4 * rows * c["KV"] * row + 4 * c["B"] * (2 + c["P"]) + (rows * c["KV"] * 12 if c["weights"] else 0),
                "flops": 0}
    if op == "evict":
        moves = 0.0
        for n in lens:
            if n > c["budget"]:
                free = c["budget"] - c["recent"]  # slots that go by weight (the few sinks aside)
                late = min(c["recent"], n - c["budget"])
                moves += late + free * (n - c["budget"] - late) / max(1, n - c["recent"])
        return {"bytes": c["KV"] * (4 * moves * row + 8 * sum(lens) + 8 * c["B"] * c["S"]) + 8 * c["B"], "flops": 0}
    moved = sum(lens) * c["moved"]  # a survivor's rows are read once however many beams take them
    read = sum(lens) * min(c["moved"], c["K"] - c["moved"])
    return {"bytes": 2 * c["layers"] * c["KV"] * row * (moved + read) + 12 * c["B"] * c["K"], "flops": 0}


# ---------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    c, s = case, prepare(case, seed)
    op = c["op"]
    if op == "attention":
        B, H, N, D = s["q"].shape
        KV = s["k"].shape[1]
        G = H // KV
        o = torch.zeros((B, H, N, D), dtype=torch.float64, device="cuda")
        w_out = None if s["weights"] is None else s["weights_out"].double()
        w_new = None if s["weights"] is None else torch.zeros((B, KV, N), dtype=torch.float64, device="cuda")
        for b, n in enumerate(s["lens"].tolist()):
            at = torch.arange(n + N, device="cuda")
            step = torch.arange(N, device="cuda") if s["depth"] is None else s["depth"][b].long()
            at[n:] = n + step
            sees = torch.ones((N, n + N), dtype=torch.bool, device="cuda")
            sees[:, n:] = torch.ones((N, N), dtype=torch.bool, device="cuda").tril() if s["tree"] is None else s["tree"][b]
            if c["window"]:
                sees &= at[None, :] - (n + step)[:, None] > -c["window"]
            for h in range(KV):
                k = torch.cat([s["k"][b, h, :n], s["k_new"][b, h]]).double().nan_to_num(0)
                v = torch.cat([s["v"][b, h, :n], s["v_new"][b, h]]).double().nan_to_num(0)
                for g in range(G):
                    x = (s["q"][b, h * G + g].double() @ k.T) * s["scale"]
                    p = torch.softmax(torch.where(sees, x, -math.inf), 1).nan_to_num(0)
                    o[b, h * G + g] = p @ v
                    if w_out is not None:
                        w_out[b, h, :n] += p[:, :n].sum(0) + (s["weights"][b, h, :n].double() if g == 0 else 0)
                        w_new[b, h] += p[:, n:].sum(0)
        return o if w_out is None else (o, w_out, w_new)
    if op == "select":
        B, K, V = s["logits"].shape
        scores = torch.full((B, c["n"]), -math.inf, dtype=torch.float64, device="cuda")
        for b in range(B):
            rows = s["logits"][b].double()
            if c["cap"]:
                rows = torch.tanh(rows / c["cap"]) * c["cap"]
            rows = torch.log_softmax(rows, 1)
            if s["finished"] is not None:
                rows[s["finished"][b]] = -math.inf
                rows[s["finished"][b], 0] = 0.0
            rows = rows + s["scores"][b].double()[:, None]
            best = torch.topk(rows.nan_to_num(-math.inf, posinf=-math.inf).flatten(), c["n"])
            scores[b] = best.values
            if c["order"] == "slot":
                beams = (best.indices // V).tolist()
                slots, free = {}, [t for t in range(K) if t not in beams]
                for rank, parent in enumerate(beams):
                    slots[parent if parent not in slots else free.pop(0)] = rank
                scores[b] = best.values[[slots[t] for t in range(K)]]
        return scores, None, None
    if op == "reorder":
        K = c["K"]
        beams, lens = s["beam"].flatten().tolist(), s["lens"].tolist()
        out = []
        for x in s["caches"]:
            y = x.clone()
            for r, parent in enumerate(beams):
                src = r - r % K + parent
                y[r, :, :lens[src]] = x[src, :, :lens[src]]
            out.append(y)
        return out
    if op == "append":
        path = s["path"].tolist() if s["path"] is not None else [list(range(c["N"]))] * c["B"]
        for b, n in enumerate(s["lens"].tolist()):
            took = path[b][:path[b].index(-1)] if -1 in path[b] else path[b]
            end = n + len(took)
            s["k"][b, :, n:end], s["v"][b, :, n:end] = s["k_new"][b][:, took], s["v_new"][b][:, took]
            if s["weights"] is not None:
                s["weights"][b, :, n:end] = s["draft_weights"][b][:, took]
        return (s["k"], s["v"], None) + ((s["weights"], None) if s["weights"] is not None else ())
    w_out = torch.zeros(s["weights"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["lens"].tolist()):
        for h in range(c["KV"]):
            w, pos = s["weights"][b, h, :n].cpu().numpy(), s["positions"][b, h, :n].cpu().numpy()
            safe = (pos < c["sink"]) | (pos > pos.max() - c["recent"])
            ranked = np.lexsort((np.arange(n), -w.astype(np.float64), ~safe))
            kept = set(ranked[:c["budget"]].tolist())
            holes = [t for t in range(min(n, c["budget"])) if t not in kept]
            came = sorted(t for t in kept if t >= c["budget"])
            src = np.arange(min(n, c["budget"]))
            src[holes] = came
            for x in (s["k"], s["v"]):
                x[b, h, holes] = x[b, h, came]
            w_out[b, h, :len(src)] = torch.from_numpy(w[src].astype(np.float64)).cuda()
    return s["k"], s["v"], w_out, None, None
