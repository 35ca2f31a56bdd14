"""What the operators of the paged 8-bit cache are timed on: giving out its pages, attention
over it, appending to it (rows become 8 bits when their page is full), and the verification
of drafted tokens that says which rows are appended.

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
# H, KV, D: query heads, cache heads, head size; P: tokens of a page; S: tokens of the longest
# sequence in the cache; N: new tokens of each sequence; `spread`: the sequences' lengths run
# from S down to (1 - spread) S; `empty`: sequences with nothing in the cache; `pad`: drafts of
# each tree that stand for nothing (their K / V rows hold whatever was in memory).
def listed():
    return [
        # One user, one token: a full-attention layer (head size 512, one cache head) behind a
        # prompt of 3658 tokens; the call's latency counts.
        dict(name="attend one token", op="attention", B=1, H=8, KV=1, D=512, P=64, S=3658, spread=0.0, empty=0, N=1,
             tree=False, pad=0, window=0, sink=0, dtype="bf16"),
        # A serving batch's decode step over ragged lengths: bound by reading the cache.
        dict(name="attend batch", op="attention", B=32, H=32, KV=8, D=128, P=64, S=8191, spread=0.75, empty=0, N=1,
             tree=False, pad=0, window=0, sink=0, dtype="bf16"),
        # Verifying trees of 24 drafts for 16 sequences: 192 query rows share each cache head.
        dict(name="attend tree of 24", op="attention", B=16, H=16, KV=2, D=256, P=32, S=4000, spread=0.5, empty=1,
             N=24, tree=True, pad=2, window=0, sink=0, dtype="bf16"),
        # A 512-row micro-batch of a prompt behind the 3146 tokens before it, on a sliding layer
        # whose first four tokens stay visible.
        dict(name="attend chunk, sliding", op="attention", B=1, H=8, KV=1, D=256, P=64, S=3146, spread=0.0, empty=0,
             N=512, tree=False, pad=0, window=512, sink=4, dtype="fp16"),
        # One token of every sequence of a small batch: a page is full now and then.
        dict(name="append one token", op="append", B=8, KV=1, D=256, P=16, S=60, N=1, path=False, spread=0.5,
             dtype="bf16"),
        # The accepted paths of drafted trees of a serving batch.
        dict(name="append paths", op="append", B=64, KV=8, D=128, P=32, S=120, N=24, path=True, spread=0.7,
             dtype="bf16"),
        # Whole prompts of ragged lengths go into the cache of one layer.
        dict(name="append prompts", op="append", B=4, KV=8, D=128, P=64, S=40, N=4000, path=False, spread=0.9,
             dtype="bf16"),
        # Pages for a token and its five drafts in a few users' caches, and back when none is taken.
        dict(name="assign 8 tables", op="assign", B=8, M=64, P=64, S=3658, room=6, spread=0.5, ended=0, window=0,
             sink=0, short=0),
        # A large server's tables on a sliding layer: the window has left pages behind, a request
        # has ended, and there are too few pages for all.
        dict(name="assign 512 tables", op="assign", B=512, M=2048, P=16, S=30000, room=64, spread=0.9, ended=1,
             window=4096, sink=4, short=400),
        # Five drafts of one user's draft model, fp32 logits of the 262144-wide head.
        dict(name="verify 5 drafts", op="verify", B=1, N=6, V=262144, tree=False, draft=True, temperature=1.0, cap=0.0,
             dtype="fp32", pad=0),
        # A batch's drafted trees, bf16 logits of the int8 head with the softcap.
        dict(name="verify 24 trees", op="verify", B=24, N=16, V=262144, tree=True, draft=True, temperature=0.8,
             cap=30.0, dtype="bf16", pad=2),
        # The same head answering greedily: drafts are taken while they are the largest logit.
        dict(name="verify greedy", op="verify", B=16, N=8, V=262144, tree=False, draft=False, temperature=0.0,
             cap=0.0, dtype="bf16", pad=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "append", "append", "assign", "verify", "verify"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    P = rng.choice([16, 32, 64, 64, 128])
    if op == "attention":
        D = rng.choice([64, 128, 256, 512])
        KV = rng.choice([1, 1, 2, 4, 8])
        G = rng.choice([1, 2, 3, 4, 5, 8])
        kind = rng.choice(["token", "token", "chain", "tree"])
        N = 1 if kind == "token" else _log(rng, 2, 64)
        B = _log(rng, 1, 48)
        # at most 64 MB of keys of one call, and 2^26 scores
        most = min(16384, (1 << 26) // (B * KV * D), (1 << 26) // (B * KV * G * N))
        S = _log(rng, 1, max(2, most))
        window = rng.choice([0, 0, 64, 300, 512])
        return dict(op=op, B=B, H=KV * G, KV=KV, D=D, P=P, S=S, spread=rng.choice([0.0, 0.5, 0.95]),
                    empty=rng.choice([0, 0, 1]) if B > 1 else 0, N=N, tree=kind == "tree",
                    pad=rng.randint(0, N // 4) if kind == "tree" else 0, window=window,
                    sink=rng.choice([0, 4, 100]) if window else 0, dtype=dtype)
    if op == "append":
        N = _log(rng, 1, 2000)
        B = min(_log(rng, 1, 64), max(1, 8000 // N))
        return dict(op=op, B=B, KV=rng.choice([1, 2, 5, 8]), D=rng.choice([64, 128, 256]), P=P, S=_log(rng, 1, 300), N=N,
                    path=N <= 64 and rng.random() < 0.5, spread=0.5, dtype=dtype)
    if op == "assign":
        B, M = _log(rng, 1, 512), _log(rng, 4, 2048)
        window = rng.choice([0, 0, 500, 4096])
        room = rng.randint(1, 64)
        return dict(op=op, B=B, M=M, P=P, S=rng.randint(1, max(1, M * P - room)), room=room, spread=rng.random(),
                    ended=rng.randint(0, B // 8), window=window, sink=rng.choice([0, 4]) if window else 0,
                    short=rng.randint(0, B))
    N, V = _log(rng, 1, 16), _log(rng, 64, 262144)
    B = min(_log(rng, 1, 24), (1 << 25) // (N * V) + 1)
    return dict(op="verify", B=B, N=N, V=V, tree=rng.random() < 0.5, draft=rng.random() < 0.6,
                temperature=rng.choice([0.0, 0.6, 1.0, 1.0, 1.5]), cap=rng.choice([0.0, 30.0]),
                dtype=rng.choice(["fp32", "bf16", "fp16"]), pad=rng.randint(0, N // 4))


# ---------------------------------------------------------------- states
def _lens(c):
    """The sequences' lengths of a case, longest first (a seed shuffles them)."""
    B, S = c["B"], c["S"]
    lens = [max(1, int(round(S * (1.0 - c["spread"] * b / max(1, B - 1))))) for b in range(B)]
    for b in range(c.get("empty", 0)):
        lens[B - 1 - b] = 0
    return lens


def _counts(c):
    """The new tokens that each sequence appends: all, or ragged where a batch is padded."""
    B, N = c["B"], c["N"]
    return [max(1, N - (N * b) // (2 * B)) for b in range(B)] if N > 1 else [1] * B


def _rows(gen, shape, dtype, scale=1.0):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).mul_(scale).to(dtype)


def _trees(rng, B, N, pad):
    """Ancestor masks, depths and parents of B random trees of N - pad drafts below draft 0."""
    mask, depth = np.zeros((B, N, N), dtype=bool), np.zeros((B, N), dtype=np.int32)
    parents = np.full((B, N), -1, dtype=np.int32)
    for b in range(B):
        for i in range(N - pad):
            if i:
                parents[b, i] = parent = int(rng.integers(max(0, i - 8), i))
                mask[b, i] = mask[b, parent]
                depth[b, i] = depth[b, parent] + 1
            mask[b, i, i] = True
    return mask, depth, parents


def _pool(gen, pages, KV, P, D):
    """Pages of an 8-bit cache as they stand after being filled, with a few strong channels."""
    x = torch.randn((pages, KV, P, D), generator=gen, device="cuda")
    x[..., :4] *= 3
    scale = x.abs().amax((2, 3)) / 127
    return torch.round(x / scale[:, :, None, None]).to(torch.int8), scale


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    s = {"case": c}
    op, B = c["op"], c["B"]

    def ints(values):
        return torch.tensor(np.asarray(values), dtype=torch.int32, device="cuda")

    if op == "verify":
        N, V, dt = c["N"], c["V"], DTYPES[c["dtype"]]
        s["logits"] = _rows(gen, (B, N, V), dt, 4.0)
        parents = _trees(rng, B, N, c["pad"])[2] if c["tree"] else np.tile(np.arange(-1, N - 1, dtype=np.int32), (B, 1))
        if c["pad"] and not c["tree"]:
            parents[:, N - c["pad"]:] = -1
        s["parent"] = ints(parents)
        up = s["parent"].long().clamp(min=0)
        s["draft"], s["tokens"] = None, torch.zeros((B, N), dtype=torch.int64, device="cuda")
        b = torch.arange(B, device="cuda")
        if c["draft"]:  # a draft model whose logits are the target's, a little off
            s["draft"] = torch.empty_like(s["logits"])
            for i in range(N):
                off = torch.randn((B, V), generator=gen, device="cuda") * 0.7
                s["draft"][:, i] = (s["logits"][:, i].float() + off).to(dt)
        for i in range(1, N):
            if c["draft"]:  # sampled from the draft model's probabilities
                off = -torch.log(-torch.log(torch.rand((B, V), generator=gen, device="cuda").clamp(1e-20, 1 - 1e-7)))
                row = s["draft"][b, up[:, i]].float() / max(c["temperature"], 1e-2)
            else:           # chosen by something cheaper
                off = torch.randn((B, V), generator=gen, device="cuda") * 0.7
                row = s["logits"][b, up[:, i]].float()
            s["tokens"][:, i] = (row + off).argmax(1)
        s["uniform"] = torch.rand((B, N), generator=gen, device="cuda")
        return s

    P = c["P"]
    lens = np.asarray(_lens(c))[rng.permutation(B)]
    if op == "assign":
        M = c["M"]
        # What an earlier step left: pages up to the sequences' lengths (all of them, windowed
        # ones too: the window has moved on), in the order in which the pool gave them out.
        held = np.minimum(-(-lens // P), M)
        pages = int(held.sum()) + B * (c["room"] // P + 2)
        ids = rng.permutation(pages).astype(np.int32)
        page = np.arange(M)[None, :]
        dead = np.maximum(lens + 1 - c["window"], 0) // P if c["window"] else np.zeros(B, dtype=np.int64)
        there = (page < held[:, None]) & ((page >= dead[:, None] - 2) | (page * P < c["sink"]))
        table = np.full((B, M), -1, dtype=np.int32)
        at = int(there.sum())
        table[there] = ids[:at]
        active = np.ones(B, dtype=bool)
        active[rng.permutation(B)[:c["ended"]]] = False
        # `short`: so many pages fewer than the step needs, with those that come back
        need = int(np.where(active, np.minimum(-(-(lens + c["room"]) // P), M) - held, 0).sum())
        back = int((there & ~(active[:, None] & ((page >= dead[:, None]) | (page * P < c["sink"])))).sum())
        top = max(0, min(pages - at, need - back - c["short"])) if c["short"] else pages - at
        free = np.full(pages, -1, dtype=np.int32)
        free[:top] = ids[at:at + top]
        s["table"], s["lens"], s["free"], s["top"] = ints(table), ints(lens), ints(free), ints([top])
        s["active"] = torch.from_numpy(active).cuda() if c["ended"] else None
        return s

    KV, D, N, dt = c["KV"], c["D"], c["N"], DTYPES[c["dtype"]]
    s["lens"] = ints(lens)
    M = -(-(int(lens.max()) + N) // P) + 1
    touched = -(-(lens + N) // P) + 1 if op == "append" else lens // P
    pages = int(touched.sum()) + 3
    ids = rng.permutation(pages - 1).astype(np.int32)  # (the pool's last page belongs to nobody)
    table = np.full((B, M), -1, dtype=np.int32)
    at = 0
    for b in range(B):
        n = min(int(touched[b]), M)
        table[b, :n] = ids[at:at + n]
        at += n
    s["table"] = ints(table)
    s["k"], s["k_scale"] = _pool(gen, pages, KV, P, D)
    s["v"], s["v_scale"] = _pool(gen, pages, KV, P, D)
    s["k_tail"], s["v_tail"] = _rows(gen, (B, KV, P, D), dt), _rows(gen, (B, KV, P, D), dt)
    s["k_new"], s["v_new"] = _rows(gen, (B, KV, N, D), dt), _rows(gen, (B, KV, N, D), dt)
    if op == "attention":
        behind = torch.arange(P, device="cuda")[None, :] >= (s["lens"] % P)[:, None]
        for name in ("k_tail", "v_tail"):  # what was in memory behind each sequence
            s[name].masked_fill_(behind[:, None, :, None], math.nan)
        # Keys of about unit mean square per element and queries that give scores of a deviation of 2.
        s["q"] = _rows(gen, (B, c["H"], N, D), dt, 2.0)
        s["scale"] = D ** -0.5
        s["tree"] = s["depth"] = None
        if c["tree"]:
            mask, depth, _ = _trees(rng, B, N, c["pad"])
            s["tree"], s["depth"] = torch.from_numpy(mask).cuda(), ints(depth)
            if c["pad"]:
                for name in ("k_new", "v_new"):
                    s[name][:, :, N - c["pad"]:] = math.nan
        return s
    counts = np.asarray(_counts(c))[rng.permutation(B)]
    s["path"] = s["count"] = None
    if c["path"]:
        path = np.full((B, N), -1)
        for b in range(B):  # from draft 0 down to some draft of the tree
            n = int(rng.integers(1, min(N, 9) + 1))
            path[b, 1:n] = np.sort(rng.permutation(N - 1)[:n - 1]) + 1
            path[b, 0] = 0
        s["path"] = ints(path)
    elif N > 1:
        s["count"] = ints(counts)
    return s


# ---------------------------------------------------------------- one pass
def _values(pages, scale):
    """What pages of 8 bits stand for."""
    return pages * scale[:, :, None, None]


def _attention(c, s):
    B, H, N, D = s["q"].shape
    KV, P = s["k"].shape[1:3]
    M, G, dev = s["table"].shape[1], H // KV, s["q"].device
    at = s["table"].long().clamp(min=0)

    def keys(name):
        old = _values(s[name][at].flatten(0, 1), s[name + "_scale"][at].flatten(0, 1))
        old = old.reshape(B, M, KV, P, D).transpose(1, 2).reshape(B, KV, M * P, D)
        return torch.cat([old, s[name + "_tail"].float(), s[name + "_new"].float()], 2)

    lens = s["lens"].long()[:, None]
    full = lens // P * P
    slot, i = torch.arange(M * P, device=dev)[None], torch.arange(N, device=dev)
    depth = i[None, :].expand(B, N) if s["depth"] is None else s["depth"].long()
    pos = torch.cat([slot.expand(B, -1), full + torch.arange(P, device=dev), lens + depth], 1)[:, None]
    there = torch.cat([slot < full, full + torch.arange(P, device=dev) < lens], 1)
    tree = (i[None, :] <= i[:, None]).expand(B, N, N) if s["tree"] is None else s["tree"]
    see = torch.cat([there[:, None].expand(B, N, -1), tree], 2)
    if c["window"]:
        see = see & ((pos > (lens + depth)[:, :, None] - c["window"]) | (pos < c["sink"]))
    used = see.any(1)[:, None, :, None]
    see = see[:, None, None].expand(B, KV, G, N, -1).reshape(B, KV, G * N, -1)
    q = s["q"].float().reshape(B, KV, G * N, D)
    x = (q @ torch.where(used, keys("k"), 0.0).transpose(2, 3) * s["scale"]).masked_fill(~see, -math.inf)
    top = x.amax(3, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(3, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    return (p @ torch.where(used, keys("v"), 0.0)).reshape(B, H, N, D).to(s["q"].dtype)


def _append(c, s):
    B, KV, P, D = s["k_tail"].shape
    N, dev = s["k_new"].shape[2], s["k"].device
    path = torch.arange(N, device=dev)[None].expand(B, N) if s["path"] is None else s["path"].long()
    if s["count"] is not None:
        path = torch.where(torch.arange(N, device=dev) < s["count"][:, None], path, -1)
    took = (path >= 0).long().cumprod(1).sum(1)
    lens = s["lens"].long()
    J = (P - 1 + N) // P + 1                                                    # pages that a sequence may reach
    first, j = lens // P, torch.arange(J, device=dev)
    at = torch.arange(J * P, device=dev)[None]
    rel = at - (lens % P)[:, None]                                              # < 0: a row of the tail
    draft = path.gather(1, rel.clamp(0, N - 1)).clamp(min=0)
    done = (first[:, None] + j + 1) * P <= (lens + took)[:, None]
    M = s["table"].shape[1]
    page = s["table"].long().gather(1, (first[:, None] + j).clamp(max=M - 1))
    # A page that is not full now gets what it holds; one that is not there stands for the pool's last.
    page = torch.where((page >= 0) & (first[:, None] + j < M), page, s["k"].shape[0] - 1)
    out = []
    for name in ("k", "v"):
        tail, new = s[name + "_tail"], s[name + "_new"]
        rows = torch.where((rel < 0)[:, None, :, None],
                           tail.gather(2, at.clamp(max=P - 1)[:, None, :, None].expand(B, KV, J * P, D)),
                           new.gather(2, draft[:, None, :, None].expand(B, KV, J * P, D)))
        x = rows.float().reshape(B, KV, J, P, D).transpose(1, 2)
        top = x.abs().amax((3, 4))
        q = torch.round(x * 127 / torch.where(top > 0, top, 1.0)[..., None, None]).to(torch.int8)
        s[name][page] = torch.where(done[:, :, None, None, None], q, s[name][page])
        s[name + "_scale"][page] = torch.where(done[:, :, None], top / 127, s[name + "_scale"][page])
        left = (lens + took) % P
        r = torch.arange(P, device=dev)[None]
        src = ((lens + took) // P - first)[:, None] * P + r
        fresh = (r < left[:, None])[:, None, :, None]
        tail.copy_(torch.where(fresh, rows.gather(2, src.clamp(max=J * P - 1)[:, None, :, None].expand(B, KV, P, D)), tail))
        out += [_values(s[name], s[name + "_scale"]), s[name + "_scale"], tail]
    return (*out, (lens + took).int())


def _assign(c, s, room):
    table, free, top = s["table"], s["free"], s["top"]
    B, M = table.shape
    i = torch.arange(M, device=table.device)[None]
    lens, P = s["lens"].long()[:, None], c["P"]
    live = torch.ones_like(lens, dtype=torch.bool) if s["active"] is None else s["active"][:, None]
    need = torch.where(live, (lens + room + P - 1) // P, 0)
    want = i < need
    if c["window"]:
        want = want & (((i + 1) * P > lens + 1 - c["window"]) | (i * P < c["sink"]))
    back = (table >= 0) & ~want
    order = (back.flatten().long().cumsum(0) - 1).reshape(B, M) + top.long()
    wide = torch.cat([free, free[:1]])                                          # one place for what does not go back
    wide.scatter_(0, torch.where(back, order, len(free)).flatten(), table.flatten())
    free.copy_(wide[:-1])
    top.add_(back.sum())
    table.masked_fill_(back, -1)
    miss = want & (table < 0) & (need <= M)
    count = miss.sum(1)
    ok = (need[:, 0] <= M) & ((count == 0) | (count.cumsum(0) <= top.long()))
    take = miss & ok[:, None]
    order = top.long() - (take.flatten().long().cumsum(0)).reshape(B, M)
    table.copy_(torch.where(take, free[order.clamp(min=0, max=len(free) - 1)], table))
    top.sub_(take.sum())
    return ok


def _verify(c, s):
    x, tokens, parent = s["logits"], s["tokens"], s["parent"]
    B, N, V = x.shape
    dev, greedy = x.device, c["temperature"] == 0
    cur = torch.zeros(B, dtype=torch.int64, device=dev)
    taken = torch.ones(B, dtype=torch.int64, device=dev)
    path = torch.full((B, N), -1, dtype=torch.int32, device=dev)
    path[:, 0] = 0
    if greedy:
        best = x.argmax(2)
    else:
        def share(t, cap):
            t = t.double()
            return torch.softmax((cap * torch.tanh(t / cap) if cap else t) / c["temperature"], 1)
        w = share(x[:, 0], c["cap"])
    for i in range(1, N):                                                       # parents come before children
        here = parent[:, i] == cur
        t = tokens[:, i:i + 1]
        if greedy:
            ok = here & (best.gather(1, cur[:, None]) == t)[:, 0]
        else:
            rows = torch.arange(B, device=dev)
            q = (torch.zeros_like(w).scatter_(1, t, 1.0) if s["draft"] is None
                 else share(s["draft"][rows, cur], 0.0))
            ok = here & (s["uniform"][:, i].double() * q.gather(1, t)[:, 0] < w.gather(1, t)[:, 0])
            rest = torch.where(q > 0, 0.0, w) if s["draft"] is None else (w - q).clamp(min=0)
            total = rest.sum(1, keepdim=True)
            rest = torch.where(total > 0, rest / torch.where(total > 0, total, 1.0), w)
            w = torch.where(ok[:, None], share(x[:, i], c["cap"]), torch.where(here[:, None], rest, w))
        path.scatter_(1, taken[:, None], torch.where(ok, i, path.gather(1, taken.clamp(max=N - 1)[:, None])[:, 0].long())
                      .int()[:, None])
        cur = torch.where(ok, i, cur)
        taken = taken + ok
    if greedy:
        return path, taken.int(), best.gather(1, cur[:, None])[:, 0]
    total = w.cumsum(1)
    over = total > s["uniform"][:, :1].double() * total[:, -1:]
    return path, taken.int(), over.int().argmax(1)


def run(state):
    s, c = state, state["case"]
    op = c["op"]
    if own:
        w8 = _kernels()
        if op == "attention":
            return w8.attention_paged(s["q"], s["k"], s["v"], s["k_scale"], s["v_scale"], s["k_tail"], s["v_tail"],
                                      s["table"], s["lens"], s["k_new"], s["v_new"], tree=s["tree"], depth=s["depth"],
                                      window=c["window"], sink=c["sink"], scale=s["scale"])
        if op == "append":
            lens = w8.paged_append(s["k"], s["v"], s["k_scale"], s["v_scale"], s["k_tail"], s["v_tail"], s["table"],
                                   s["lens"], s["k_new"], s["v_new"], path=s["path"], count=s["count"])
            return (_values(s["k"], s["k_scale"]), s["k_scale"], s["k_tail"], _values(s["v"], s["v_scale"]),
                    s["v_scale"], s["v_tail"], lens)
        if op == "assign":  # pages for the step's new tokens; none is taken, so that they go back
            ok = w8.page_assign(s["table"], s["lens"], s["free"], s["top"], c["P"], room=c["room"], active=s["active"],
                                window=c["window"], sink=c["sink"])
            table = s["table"].clone()
            back = w8.page_assign(s["table"], s["lens"], s["free"], s["top"], c["P"], room=0, active=s["active"],
                                  window=c["window"], sink=c["sink"])
            return ok, table, back, s["table"], s["free"], s["top"]
        return w8.draft_verify(s["logits"], s["tokens"], s["uniform"], parent=s["parent"], draft=s["draft"],
                               temperature=c["temperature"], cap=c["cap"])
    if op == "attention":
        return _attention(c, s)
    if op == "append":
        return _append(c, s)
    if op == "assign":
        ok = _assign(c, s, c["room"])
        table = s["table"].clone()
        return ok, table, _assign(c, s, 0), s["table"], s["free"], s["top"]
    return _verify(c, s)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    c = case
    op, B = c["op"], c["B"]
    if op == "verify":
        size = 4 if c["dtype"] == "fp32" else 2
        rows = B * c["N"] * (2 if c["draft"] and c["temperature"] else 1)
        return {"bytes": rows * c["V"] * size + B * c["N"] * 20 + 12 * B, "flops": 4.0 * rows * c["V"]}
    lens = _lens(c)
    if op == "assign":
        return {"bytes": 2 * 4 * B * c["M"] + 2 * 9 * B, "flops": 0}
    KV, D, P, N = c["KV"], c["D"], c["P"], c["N"]
    if op == "attention":
        W, G = c["window"], c["H"] // KV
        keys = sum(min(n, W + N - 2 + c["sink"]) if W else n for n in lens)
        pairs = sum((min(n, W - 1 + c["sink"]) if W else n) * N for n in lens) + B * N * (1 if N == 1 else N / 2)
        tail = sum(min(n, n % P) for n in lens)
        by = KV * 2 * D * ((keys - tail) + 2 * tail + 2 * B * N) + 8 * KV * keys / P + 4 * B * c["H"] * N * D
        by += 4 * B + 4 * keys / P + (B * N * N if c["tree"] else 0)
        return {"bytes": by, "flops": 4.0 * KV * G * D * pairs}
    took = [min(4.5, (min(N, 9) + 1) / 2)] * B if c["path"] else _counts(c)
    by = 0.0
    for n, m in zip(lens, took):
        done = (n % P + m) // P
        by += m * 4 * D                                   # the new rows, read (K and V, 2 bytes)
        by += done * 2 * D * P + min(done, 1) * (n % P) * 4 * D   # full pages, and the tail's rows in the first
        by += ((n + m) % P if done else m) * 4 * D        # rows that stay in the tail
    return {"bytes": KV * by + 8 * B, "flops": 0}


# ---------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    c, s = case, prepare(case, seed)
    op = c["op"]
    if op in ("assign", "verify"):
        return None  # whole numbers and truth values only
    P = c["P"]
    if op == "attention":
        B, H, N, D = s["q"].shape
        KV = s["k"].shape[1]
        o = torch.zeros((B, H, N, D), dtype=torch.float64, device="cuda")
        for b, n in enumerate(s["lens"].tolist()):
            step = torch.arange(N, device="cuda") if s["depth"] is None else s["depth"][b].long()
            at = torch.cat([torch.arange(n, device="cuda"), n + step])
            sees = torch.ones((N, n + N), dtype=torch.bool, device="cuda")
            sees[:, n:] = torch.ones((N, N), dtype=torch.bool, device="cuda").tril() if s["tree"] is None else s["tree"][b]
            if c["window"]:
                sees &= (at[None, :] - (n + step)[:, None] > -c["window"]) | (at[None, :] < c["sink"])
            ids = s["table"][b, :n // P].long()
            for h in range(KV):
                kv = []
                for name in ("k", "v"):
                    old = (s[name][ids, h].double() * s[name + "_scale"][ids, h].double()[:, None, None]).reshape(-1, D)
                    kv.append(torch.cat([old, s[name + "_tail"][b, h, :n % P].double(),
                                         s[name + "_new"][b, h].double()]).nan_to_num(0))
                for g in range(h * H // KV, (h + 1) * H // KV):
                    x = (s["q"][b, g].double() @ kv[0].T) * s["scale"]
                    o[b, g] = torch.softmax(torch.where(sees, x, -math.inf), 1).nan_to_num(0) @ kv[1]
        return o
    out = []
    for name in ("k", "v"):
        old, scale, tail = s[name], s[name + "_scale"].double(), s[name + "_tail"].double()
        values = old.double() * scale[:, :, None, None]
        for b, n in enumerate(s["lens"].tolist()):
            order = list(range(c["N"])) if s["path"] is None else [i for i in s["path"][b].tolist() if i >= 0]
            if s["count"] is not None:
                order = order[:int(s["count"][b])]
            rows = torch.cat([tail[b, :, :n % P], s[name + "_new"][b][:, order].double()], 1)
            for j in range(rows.shape[1] // P):
                page = int(s["table"][b, n // P + j])
                part = rows[:, j * P:(j + 1) * P]
                most = part.abs().amax((1, 2))
                scale[page] = most / 127
                values[page] = torch.round(part * 127 / most[:, None, None]) * scale[page][:, None, None]
            rest = rows.shape[1] % P
            tail[b, :, :rest] = rows[:, rows.shape[1] - rest:]
        out += [values, scale, tail]
    return (*out, None)
