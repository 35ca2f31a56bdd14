"""The operators of the paged 8-bit cache and draft verification against plain 64-bit definitions.

Tolerances.  Appended pages, tables, paths and tokens are equal bit for bit.  Attention: with u =
half a step of the 16-bit type (2^-8 bf16, 2^-11 fp16; where pages' weights are rounded to fp16
that is less), each weight is rounded once (u p_j) and the output once (u |o|).  A weight of a
page's key is held relative to the largest scale of V, down to 2^-25 against a sum of 2^7: 2^-31 of
the largest |v| a key.  Scores: keys of pages are multiplied as 1152 + k8, whose excess a start value
takes off, in D / 8 steps of fp32 sums (the matrix instructions add 8 or 16 products at a time) of at most 2432
sum |q| ks scale, 2^-23 of it each; 16-bit keys as fp32 sums of D + 4 terms; and an argument x of exp2
is off by 2^-21 |x| + 2^-18 (its scale and, on the tensor cores' schedule, the logarithm of V's scale).
An error e of a score moves a probability and the sum it is divided by by 2 e: |out - o| <=
(u + 2 e) sum p|v| + u |o| + 2^-31 n max|v| (+ 2^-20 sum p|v| for the fp32 sums).
"""
import math
import random

import pytest
import torch

import gemma_npu_b200 as w8

pytestmark = pytest.mark.gpu
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])


def rows(gen, shape, dt, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dt)


def cache(seed, KV, D, P, lens, dt=torch.bfloat16, layout="head", spare=3, spread=0.0, M=None):
    """A paged cache of sequences of these lengths: dict of its tensors.  What belongs to nobody is
    NaN (tail rows behind a length, scales of unused pages) or -1 (table entries)."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    B, full = len(lens), [n // P for n in lens]
    pages = sum(full) + spare
    if layout == "head":
        k, v = (torch.randint(-127, 128, (pages, KV, P, D), generator=gen, device="cuda", dtype=torch.int8) for _ in range(2))
        kt, vt = (rows(gen, (B, KV, P, D), dt) for _ in range(2))
    else:  # token-major pages and tails, slices of wider buffers
        k, v = (torch.randint(-127, 128, (pages, P, KV + 1, D + 16), generator=gen, device="cuda", dtype=torch.int8)
                [:, :, 1:, 16:].transpose(1, 2) for _ in range(2))
        kt, vt = (rows(gen, (B, P, KV, D + 8), dt)[..., 8:].transpose(1, 2) for _ in range(2))
    ks, vs = (torch.rand((pages, KV), generator=gen, device="cuda") * 0.01 + 0.02 for _ in range(2))
    if spread:
        vs *= torch.exp(spread * torch.randn((pages, KV), generator=gen, device="cuda"))
    if layout != "head":
        ks, vs = (torch.stack([s, s * 0 + math.nan], 2)[..., 0] for s in (ks, vs))
    ids = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    M = max(full + [1]) + 1 if M is None else M
    table = torch.full((B, M + 3), -1, dtype=torch.int32)[:, :M]
    at = 0
    for b in range(B):
        table[b, :full[b]] = torch.tensor(ids[at:at + full[b]], dtype=torch.int32)
        at += full[b]
        kt[b, :, lens[b] % P:] = math.nan
        vt[b, :, lens[b] % P:] = math.nan
    for p in ids[at:]:
        ks[p] = math.nan
        vs[p] = math.nan
    return dict(k=k, v=v, k_scale=ks, v_scale=vs, k_tail=kt, v_tail=vt, table=table.cuda(),
                lens=torch.tensor(lens, dtype=torch.int32, device="cuda"))


def new(seed, B, H, KV, D, N, dt):
    gen = torch.Generator(device="cuda").manual_seed(seed + 1000)
    return rows(gen, (B, H, N, D), dt, 2.0), rows(gen, (B, KV, N, D), dt), rows(gen, (B, KV, N, D), dt)


def tree_of(seed, B, N, pad=0):
    g = torch.Generator().manual_seed(seed)
    mask, depth = torch.zeros((B, N, N), dtype=torch.bool), torch.zeros((B, N), dtype=torch.int32)
    parent = torch.full((B, N), -1, dtype=torch.int32)
    for b in range(B):
        for i in range(N - pad):
            p = int(torch.randint(max(0, i - 6), i, (1,), generator=g)) if i else -1
            parent[b, i] = p
            if p >= 0:
                mask[b, i] = mask[b, p]
                depth[b, i] = depth[b, p] + 1
            mask[b, i, i] = True
    return mask.cuda(), depth.cuda(), parent.cuda()


def want_attention(c, q, kn, vn, tree=None, depth=None, window=0, sink=0, scale=1.0):
    """(out, its tolerance without u, sum p|v|) in 64 bits."""
    B, H, N, D = q.shape
    KV, P = c["k"].shape[1:3]
    G = H // KV
    o, tol, pv = (torch.zeros((B, H, N, D), dtype=torch.float64, device="cuda") for _ in range(3))
    for b, n in enumerate(c["lens"].tolist()):
        step = torch.arange(N, device="cuda") if depth is None else (depth if depth.dim() == 1 else depth[b]).long()
        own = torch.ones((N, N), dtype=torch.bool, device="cuda").tril() if tree is None else (
            tree if tree.dim() == 2 else tree[b])
        sees = torch.cat([torch.ones((N, n), dtype=torch.bool, device="cuda"), own], 1)
        if window:
            at = torch.cat([torch.arange(n, device="cuda"), n + step])
            sees &= (at[None] > (n + step)[:, None] - window) | (at[None] < sink)
        ids, f = c["table"][b, :n // P].long(), n // P * P
        there = ids >= 0  # (pages before a window may be gone)
        ids = ids.clamp(min=0)
        some = sees.any(0)
        for h in range(H):
            kv = []
            for x, xn in (("k", kn), ("v", vn)):
                old = c[x][ids, h // G].double() * c[x + "_scale"][ids, h // G].double()[:, None, None]
                old[~there] = 0
                kv.append(torch.cat([old.reshape(-1, D), c[x + "_tail"][b, h // G, :n - f].double(), xn[b, h // G].double()]))
            keys, vals = kv
            keys[~some], vals[~some] = 0, 0
            x = q[b, h].double() @ keys.T * scale
            p = torch.softmax(x.masked_fill(~sees, -math.inf), 1)
            p = torch.where(sees.any(1, keepdim=True), p, 0.0)
            e = (D + 4) * 2.0 ** -24 * (q[b, h].double().abs() @ keys.abs().T * scale) + 2.0 ** -21 * x.abs() + 2.0 ** -18
            ks = c["k_scale"][ids, h // G].double().nan_to_num(0).repeat_interleave(P)
            e[:, :f] += D / 8 * 2.0 ** -23 * 2432 * scale * q[b, h].double().abs().sum(1, keepdim=True) * ks
            e = torch.where(sees, e, 0.0).nan_to_num(0).amax(1, keepdim=True)
            for i in range(N):  # each row adds only what it sees (0 * inf never happens)
                s = sees[i]
                o[b, h, i] = p[i, s] @ vals[s]
                pv[b, h, i] = p[i, s] @ vals[s].abs()
            tol[b, h] = (2 * e + 2.0 ** -20) * pv[b, h]
            if f:
                tol[b, h] += 2.0 ** -31 * n * float(vals[:f].abs().nan_to_num(0).max())
    return o, tol, pv


def check_out(got, want, dt):
    o, tol, pv = want
    bound = HALF[dt] * (pv + o.abs()) + tol + 1e-30 + (2.0 ** -24 if dt == torch.float16 else 0)
    err = (got.double() - o).abs()
    assert bool((err <= bound).all()), float((err - bound).max())


def attend(c, q, kn, vn, **kw):
    return w8.attention_paged(q, c["k"], c["v"], c["k_scale"], c["v_scale"], c["k_tail"], c["v_tail"], c["table"], c["lens"],
                              kn, vn, **kw)


# (H, KV, D, P, N, lens, window, sink): one token; lengths around pages and zero; groups of 1 to 8 and odd
# ones; chunks within and across tiles; windows shorter and longer than the cache, sinks in every kind of row.
SHAPES = [
    (8, 1, 512, 64, 1, [3658], 0, 0),
    (8, 1, 256, 64, 1, [3658], 512, 4),
    (4, 2, 128, 32, 1, [0, 1, 31, 32, 33, 127, 128, 129, 255, 256, 257], 0, 0),
    (4, 2, 128, 32, 1, [0, 1, 31, 32, 33, 127, 128, 129, 255, 256, 257], 7, 3),
    (5, 1, 64, 16, 1, [200, 77, 1, 16], 0, 0),
    (3, 3, 64, 128, 3, [70, 5, 300], 0, 0),
    (6, 2, 128, 16, 3, [300, 129], 64, 20),
    (9, 1, 256, 128, 1, [500, 128, 129], 0, 0),
    (16, 1, 128, 64, 1, [700, 64], 100, 70),
    (8, 8, 512, 16, 5, [64, 100], 33, 17),
    (8, 1, 512, 128, 1, [260, 383], 128, 200),
    (2, 1, 64, 16, 1, [0], 0, 0),
    (4, 1, 128, 16, 2, [0], 0, 0),
    (32, 8, 128, 16, 1, [(7 * i) % 101 for i in range(40)], 0, 0),
    # tiles dealt over CTAs, more pairs than a CTA has threads
    (64, 8, 128, 64, 1, [3000, 1, 700, 2999, 128, 129, 0, 2000, 64, 1500], 0, 0),
    (64, 8, 64, 32, 1, [3000, 1, 700, 2999, 256, 257, 0, 2000, 64, 1500], 900, 40),
    (12, 2, 512, 64, 1, [2000, 3, 1111], 0, 0),
    (4, 2, 128, 16, 1, [(37 * i) % 301 for i in range(300)], 100, 0),
    # many rows: tcgen05, whole and odd groups, splits, windows, empty caches
    (8, 1, 256, 64, 70, [131], 100, 5),
    (8, 1, 256, 64, 300, [600], 512, 4),
    (16, 2, 256, 32, 33, [500, 64], 0, 0),
    (8, 2, 128, 16, 40, [2500, 1222, 31], 0, 0),
    (6, 2, 256, 128, 50, [2900], 0, 0),
    (8, 1, 256, 16, 64, [0], 0, 0),
    (8, 1, 512, 64, 20, [260, 1000], 128, 150),
    (16, 1, 512, 16, 3, [0, 90], 2, 1),
    (8, 1, 64, 64, 100, [600, 0], 512, 130),
    (16, 2, 64, 32, 40, [300, 0, 1, 127, 128, 129, 255, 256, 257], 50, 200),
    (33, 1, 64, 128, 1, [650], 0, 0),
    (17, 1, 128, 128, 1, [650, 127, 128], 300, 129),
    # the same sizes' neighbours: several tiles of 16 (or 8) rows, and one row more than those take
    (8, 1, 512, 128, 3, [700, 0, 129], 0, 0),
    (4, 1, 512, 16, 5, [300, 64], 40, 17),
    (25, 1, 512, 32, 1, [333, 1], 0, 0),
    (12, 2, 128, 32, 8, [700, 33, 0], 0, 0),
    (7, 1, 128, 64, 7, [500, 64], 130, 70),
    (16, 2, 64, 16, 8, [600, 15, 17], 60, 33),
    (13, 1, 64, 128, 5, [520], 0, 0),
    (16, 8, 64, 32, 20, [3000, 1, 700, 2999, 256, 257, 0, 2000, 64, 1500], 900, 40),
]


@DTYPES
@pytest.mark.parametrize("shape", SHAPES, ids=[str(i) for i in range(len(SHAPES))])
def test_attention_chain(cuda, shape, dt):
    H, KV, D, P, N, lens, window, sink = shape
    c = cache(D + N, KV, D, P, lens, dt)
    a = new(P, len(lens), H, KV, D, N, dt)
    kw = dict(window=window, sink=sink, scale=D ** -0.5)
    check_out(attend(c, *a, **kw), want_attention(c, *a, **kw), dt)
    assert w8.device_status() == 0


@DTYPES
@pytest.mark.parametrize("shape", [(4, 2, 128, 32, 5, [100, 0, 33], 0, 0), (2, 1, 256, 64, 7, [300, 64], 50, 4),
                                   (8, 2, 256, 32, 24, [700, 0, 95], 0, 0), (8, 1, 512, 16, 30, [300, 17], 40, 10),
                                   (4, 1, 64, 128, 60, [500], 100, 600), (4, 4, 64, 16, 13, [100, 5], 9, 104),
                                   (4, 1, 64, 16, 13, [300, 5, 0], 9, 104), (8, 2, 128, 64, 11, [700, 64], 0, 0),
                                   (4, 2, 512, 32, 9, [200, 31], 20, 210)],
                         ids=[str(i) for i in range(9)])
def test_attention_tree(cuda, shape, dt):
    """Drafted trees: ancestors' masks, depths, sinks among the new tokens, padding drafts of NaN."""
    H, KV, D, P, N, lens, window, sink = shape
    c = cache(N, KV, D, P, lens, dt)
    q, kn, vn = new(P, len(lens), H, KV, D, N, dt)
    tree, depth, _ = tree_of(N, len(lens), N, pad=2)
    kn[:, :, N - 2:], vn[:, :, N - 2:] = math.nan, math.nan
    kw = dict(tree=tree, depth=depth, window=window, sink=sink, scale=D ** -0.5)
    check_out(attend(c, q, kn, vn, **kw), want_attention(c, q, kn, vn, **kw), dt)
    kw = dict(tree=tree[0], depth=depth[0], window=window, sink=sink, scale=D ** -0.5)  # one for all sequences
    check_out(attend(c, q, kn, vn, **kw), want_attention(c, q, kn, vn, **kw), dt)
    assert w8.device_status() == 0


@pytest.mark.parametrize("H,N", [(2, 1), (16, 1), (8, 40)])
@pytest.mark.parametrize("D,P", [(64, 16), (128, 128), (256, 32), (512, 64)])
def test_attention_strides(cuda, H, N, D, P):
    """Token-major pages and tails, slices of wider buffers, strided tables and outputs."""
    lens = [400, 3, P, 2 * P + 1]
    c = cache(D, 2, D, P, lens, layout="token")
    q, kn, vn = new(P, 4, H, 2, D, N, torch.bfloat16)
    q = q.transpose(1, 2).contiguous().transpose(1, 2)
    kn = torch.cat([kn, kn], 3)[..., :D]
    out = torch.full((4, N, H, D + 8), 7.0, device="cuda", dtype=torch.bfloat16)
    got = attend(c, q, kn, vn, scale=D ** -0.5, out=out[..., :D].transpose(1, 2))
    check_out(got, want_attention(c, q, kn, vn, scale=D ** -0.5), torch.bfloat16)
    assert got.data_ptr() == out.data_ptr() and bool((out[..., D:] == 7).all())


@pytest.mark.parametrize("H,N", [(4, 1), (8, 5), (8, 20)])
@DTYPES
def test_attention_scales_far_apart(cuda, H, N, dt):
    """Pages whose scales of V differ by orders of magnitude (O's unit moves), pages of zeros, and a zero
    scale."""
    c = cache(3, 1, 128, 16, [1000, 40], dt, spread=4.0)
    ids = c["table"][0].long()
    c["v"][ids[5]] = 0
    c["k"][ids[6]] = 0
    c["k_scale"][ids[7]] = 0
    c["v_scale"][ids[8]] = 0
    c["k_scale"][ids[9]] = c["v_scale"][ids[9]] = 0
    c["v_scale"][ids[0]] = 1e-20
    a = new(4, 2, H, 1, 128, N, dt)
    want = want_attention(c, *a, scale=0.05)
    if dt == torch.float16:  # (the output must fit)
        c["v_scale"][torch.isfinite(c["v_scale"])] /= 1 + float(want[0].abs().max()) / 100
        want = want_attention(c, *a, scale=0.05)
    check_out(attend(c, *a, scale=0.05), want, dt)


@pytest.mark.parametrize("D,KV,H,N", [(64, 1, 8, 1), (128, 2, 8, 1), (256, 1, 8, 1), (512, 1, 8, 1), (512, 1, 16, 2), (256, 1, 16, 16)])
@DTYPES
def test_attention_of_queries_off_zero(cuda, D, KV, H, N, dt):
    """Queries whose elements have a common offset, up to one sign: what pages' keys are raised by, times
    the queries' sums, has to cancel.  Scores lose more there than about 0, within the bound above; calls
    repeat to the bit."""
    c = cache(1, KV, D, 64, [1500, 700], dt)
    q, kn, vn = new(2, 2, H, KV, D, N, dt)
    for off in (1.0, 4.0, -30.0):
        x = (q.float() / 2 + off).to(dt)
        scale = D ** -0.5 / (1 + abs(off) / 8)
        got = attend(c, x, kn, vn, scale=scale)
        check_out(got, want_attention(c, x, kn, vn, scale=scale), dt)
        assert torch.equal(got, attend(c, x, kn, vn, scale=scale))


@pytest.mark.parametrize("D,KV,H,N,lens", [(64, 2, 4, 1, [100, 40, 3]), (128, 1, 8, 2, [1000, 40, 3]), (256, 2, 4, 3, [300, 48, 0]),
                                           (512, 1, 8, 1, [700, 64, 3]), (128, 8, 64, 1, [3000, 700, 2999, 128]),
                                           (128, 1, 8, 20, [1000, 40, 3])])
@pytest.mark.parametrize("size", [1e-37, 2.0 ** -125, 2.0 ** -126, 2.0 ** -127, 1e-39, 0.0])
def test_attention_of_tiny_scales(cuda, size, D, KV, H, N, lens):
    """Pages of values so small that their scales are at or below fp32's smallest normal number (what
    `paged_append` makes of bf16 rows below 1.5e-36): next to nothing is added to the other rows."""
    c = cache(4, KV, D, 16, lens)
    a = new(5, len(lens), H, KV, D, N, torch.bfloat16)
    c["v_scale"][torch.isfinite(c["v_scale"])] = size
    check_out(attend(c, *a, scale=0.05), want_attention(c, *a, scale=0.05), torch.bfloat16)
    c["v_scale"][c["table"][0, 0].long()] = 0.02  # (one page that is not)
    check_out(attend(c, *a, scale=0.05), want_attention(c, *a, scale=0.05), torch.bfloat16)


@pytest.mark.parametrize("H,N", [(4, 1), (8, 5), (8, 20)])
def test_attention_of_a_page_with_nan_scales(cuda, H, N):
    """A NaN scale is for the rows that see the page: a window keeps it from others."""
    c = cache(5, 1, 64, 16, [100, 100])
    page = int(c["table"][0, 2])  # positions 32 .. 47 of the first sequence
    a = new(6, 2, H, 1, 64, N, torch.bfloat16)
    for name in ("k_scale", "v_scale"):
        d = dict(c, **{name: c[name].clone()})
        d[name][page] = math.nan
        got = attend(d, *a, scale=0.1)
        assert bool(got[0].isnan().all()) and not bool(got[1].isnan().any()), name
        kw = dict(window=40, sink=16, scale=0.1)
        check_out(attend(d, *a, **kw), want_attention(c, *a, **kw), torch.bfloat16)


@pytest.mark.parametrize("H,N", [(4, 1), (8, 5), (8, 20)])
def test_attention_new_values_that_some_rows_see(cuda, H, N):
    """Infinite and NaN values of a new token reach the rows that see it and no others."""
    c = cache(7, 1, 128, 32, [70])
    q, kn, vn = new(8, 1, H, 1, 128, max(N, 3), torch.bfloat16)
    vn[0, 0, 1, 5], vn[0, 0, 2, 9] = math.inf, math.nan
    got = attend(c, q, kn, vn, scale=0.1)
    clean = attend(c, q, kn, vn.nan_to_num(0, 0, 0), scale=0.1)
    assert bool(got[:, :, 0].eq(clean[:, :, 0]).all())
    assert bool((got[:, :, 1:, 5] == math.inf).all()) and bool(got[:, :, 2:, 9].isnan().all())
    rest = [i for i in range(128) if i not in (5, 9)]
    assert bool(got[..., rest].eq(clean[..., rest]).all())


@pytest.mark.parametrize("H,N", [(4, 1), (8, 5), (8, 20)])
def test_attention_pages_before_the_window_may_be_gone(cuda, H, N):
    c = cache(9, 1, 64, 16, [500, 37])
    a = new(10, 2, H, 1, 64, N, torch.bfloat16)
    kw = dict(window=64, sink=20, scale=0.125)
    want = want_attention(c, *a, **kw)
    c["table"][0, 2:(500 - 63) // 16] = -1  # (the sinks' two pages stay)
    c["table"][0, 40:] = 10 ** 6            # behind the length
    check_out(attend(c, *a, **kw), want, torch.bfloat16)
    assert w8.device_status() == 0


@pytest.mark.parametrize("H,N", [(4, 1), (8, 5), (8, 20)])
@pytest.mark.parametrize("entry", [-1, 10 ** 6])
def test_attention_reports_a_missing_page(cuda, H, N, entry):
    c = cache(11, 1, 64, 16, [200])
    a = new(12, 1, H, 1, 64, N, torch.bfloat16)
    c["table"][0, 3] = entry
    got = attend(c, *a, scale=0.125)
    with pytest.raises(w8._lib.W8InvalidArgument, match="attention"):
        w8.device_status()
    assert w8.device_status() == 0 and bool(got.isfinite().all())


def test_attention_lengths_out_of_range(cuda):
    c = cache(13, 1, 64, 16, [100, 100])
    a = new(14, 2, 4, 1, 64, 1, torch.bfloat16)
    c["lens"].copy_(torch.tensor([-5, 100]))
    got = attend(c, *a, scale=0.125)
    with pytest.raises(w8._lib.W8InvalidArgument):
        w8.device_status()
    c["lens"].copy_(torch.tensor([0, 100]))
    assert bool(got.eq(attend(c, *a, scale=0.125)).all()) and w8.device_status() == 0


@pytest.mark.parametrize("H,N", [(2, 2), (6, 4)])
def test_attention_scores_far_below_zero(cuda, H, N):
    """Few rows, scores of -2^106 and less, powers of two that fp32 holds: the largest have all the weight."""
    D, P, lens = 64, 16, [37, 20]
    c = cache(3, 2, D, P, lens)
    q, kn, vn = new(3, 2, H, 2, D, N, torch.bfloat16)
    q[:] = 2.0 ** 60
    for x in ("k", "k_tail"):
        c[x][:] = (-(2 ** (torch.arange(P, device="cuda") % 5)))[:, None].to(c[x].dtype)
    c["k_tail"] *= 2.0 ** 40
    c["k_scale"][:] = 2.0 ** 40
    kn[:] = -2.0 ** 41
    o, _, pv = want_attention(c, q, kn, vn)
    check_out(attend(c, q, kn, vn), (o, 2.0 ** -20 * pv + 2.0 ** -18 * float(pv.max()), pv), torch.bfloat16)


def test_attention_offsets_beyond_32_bits(cuda):
    """A pool of more than 2^31 bytes, its last pages in use."""
    pages, P, D = 66000, 128, 256
    c = cache(15, 1, D, P, [5 * P + 3])
    pool = {x: torch.zeros((pages, 1, P, D), dtype=torch.int8, device="cuda") for x in ("k", "v")}
    ids = c["table"][0, :5].long()
    want_c = dict(c)
    at = torch.arange(pages - 5, pages, device="cuda")
    for x in ("k", "v"):
        pool[x][at] = c[x][ids]
        c[x + "_scale"] = torch.zeros((pages, 1), device="cuda").index_copy(0, at, c[x + "_scale"][ids])
    big = dict(c, k=pool["k"], v=pool["v"], table=c["table"].clone())
    big["table"][0, :5] = at.int()
    want_c["k_scale"], want_c["v_scale"] = c["k_scale"][at].index_copy(0, torch.arange(5, device="cuda"), c["k_scale"][at]), c["v_scale"][at]
    want_c = dict(want_c, k=pool["k"][at], v=pool["v"][at], table=torch.tensor([[0, 1, 2, 3, 4, -1]], device="cuda", dtype=torch.int32))
    for H, N in ((4, 1), (8, 5)):
        a = new(16, 1, H, 1, D, N, torch.bfloat16)
        assert bool(attend(big, *a, scale=0.0625).eq(attend(want_c, *a, scale=0.0625)).all())


@pytest.mark.parametrize("H,N", [(8, 1), (8, 20)])
def test_attention_repeats_itself_on_streams_and_in_graphs(cuda, H, N):
    """The same bits again, on two streams at once and captured; graphs share nothing."""
    cases = [(cache(s, 2, 128, 32, [900, 0, 333]), new(s, 3, H, 2, 128, N, torch.float16)) for s in (1, 2)]
    cases = [(cache(s, 2, 128, 32, [900, 0, 333], torch.float16), a) for s, (_, a) in zip((1, 2), cases)]
    want = [attend(c, *a, scale=0.1) for c, a in cases]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        got = []
        for s, (c, a) in zip(streams, cases):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(attend(c, *a, scale=0.1))
        torch.cuda.synchronize()
        for g, x in zip(got, want):
            assert bool(g.eq(x).all())
    graphs = []
    for c, a in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = attend(c, *a, scale=0.1)
        graphs.append((g, out))
    for _ in range(2):
        for g, out in graphs:
            out.zero_()
            g.replay()
    torch.cuda.synchronize()
    for (g, out), x in zip(graphs, want):
        assert bool(out.eq(x).all())


def test_attention_of_nothing(cuda):
    c = cache(1, 1, 64, 16, [40])
    q, kn, vn = new(1, 1, 4, 1, 64, 0, torch.bfloat16)
    assert attend(c, q, kn, vn).shape == (1, 4, 0, 64)


def test_attention_refuses(cuda):
    c = cache(1, 1, 64, 16, [40])
    q, kn, vn = new(1, 1, 4, 1, 64, 2, torch.bfloat16)
    for kw, match in ((dict(sink=3), "window"), (dict(window=4, tree=torch.ones((2, 2), dtype=torch.bool, device="cuda")), "depths"),
                      (dict(scale=0.0), "scale"), (dict(out=q), "out must not"), (dict(out=torch.empty_like(q)[:, :1]), "shape")):
        with pytest.raises(ValueError, match=match):
            attend(c, q, kn, vn, **kw)
    for change, match in ((dict(k=c["k"].float()), "k must be"), (dict(k_scale=c["k_scale"].half()), "k_scale"),
                          (dict(k_tail=c["k_tail"].half()), "k_tail"), (dict(table=c["table"].long()), "table"),
                          (dict(v_scale=c["v_scale"][:-1]), "v_scale"), (dict(lens=c["lens"].cpu()), "lens"),
                          (dict(v=c["v"][:-1]), "shape of k"), (dict(table=c["table"][:, :0].t()), "table")):
        with pytest.raises(ValueError, match=match):
            attend(dict(c, **change), q, kn, vn)
    with pytest.raises(ValueError, match="positive"):
        attend(c, q, kn[:, :, :1].expand(-1, -1, 2, -1), vn)
    with pytest.raises(w8.W8Error):
        attend({n: t[:, :, :8] if t.dim() == 4 else t for n, t in c.items()}, q, kn, vn)


# ---------------------------------------------------------------- append
def want_append(c, kn, vn, path=None, count=None):
    """The cache after appending, row by row, in exact arithmetic where bits are decided."""
    c = {n: t.clone() for n, t in c.items()}
    P = c["k"].shape[2]
    for b, n in enumerate(c["lens"].tolist()):
        order = list(range(kn.shape[2])) if path is None else path[b].tolist()
        order = order[:next((i for i, x in enumerate(order) if x < 0), len(order))]
        if count is not None:
            order = order[:int(count[b])]
        order = order[:c["table"].shape[1] * P - n]
        for x, xn in (("k", kn), ("v", vn)):
            fresh = torch.stack([xn[b, :, i] if i < kn.shape[2] else torch.zeros_like(xn[b, :, 0]) for i in order], 1) if order else xn[b, :, :0]
            all_rows = torch.cat([c[x + "_tail"][b, :, :n % P], fresh], 1)
            for j in range(all_rows.shape[1] // P):
                page = int(c["table"][b, n // P + j])
                if not 0 <= page < c["k"].shape[0]:
                    continue
                part = all_rows[:, j * P:(j + 1) * P].double()
                most = part.abs().amax((1, 2))
                fine = most.isfinite()
                q = torch.round(part.nan_to_num(0, 0, 0) * 127 / torch.where(fine & (most > 0), most, 1.0)[:, None, None])
                c[x][page] = torch.where(fine[:, None, None], q, 0.0).to(torch.int8)
                scale = (most.float().cpu() / torch.tensor(127.0)).cuda()
                c[x + "_scale"][page] = torch.where(fine, scale, torch.full_like(scale, math.nan))
            rest = all_rows.shape[1] % P
            if all_rows.shape[1] >= P:
                c[x + "_tail"][b, :, :rest] = all_rows[:, all_rows.shape[1] - rest:]
            else:
                c[x + "_tail"][b, :, :rest] = all_rows
        c["lens"][b] = n + len(order)
    return c


def give_pages(c, n):
    """Pages for n more positions of every sequence."""
    P = c["k"].shape[2]
    used = set(c["table"].flatten().tolist())
    spare = [p for p in range(c["k"].shape[0]) if p not in used]
    for b, m in enumerate(c["lens"].tolist()):
        for i in range(m // P, min(-(-(m + n) // P), c["table"].shape[1])):
            c["table"][b, i] = spare.pop()
    return c


def same(a, b):
    return bool(((a == b) | (a.isnan() & b.isnan())).all()) if a.is_floating_point() else bool(a.eq(b).all())


def run_append(c, kn, vn, **kw):
    got = {n: t.clone() for n, t in c.items()}
    got["lens"] = w8.paged_append(got["k"], got["v"], got["k_scale"], got["v_scale"], got["k_tail"], got["v_tail"], got["table"],
                                  c["lens"], kn, vn, **kw)
    return got


def check_append(c, kn, vn, **kw):
    got, want = run_append(c, kn, vn, **kw), want_append(c, kn, vn, **kw)
    for name in want:
        assert same(got[name], want[name]), name


@DTYPES
@pytest.mark.parametrize("KV,D,P,N,lens", [
    (1, 256, 16, 1, [0, 1, 14, 15, 16, 31]), (2, 128, 64, 1, [63, 64, 5]), (3, 64, 32, 7, [0, 25, 26, 31, 32]),
    (1, 512, 128, 130, [0, 1, 126, 127, 128]), (8, 128, 64, 300, [40, 0, 63]), (1, 64, 16, 100, [9]),
    (2, 256, 128, 3, [125, 124, 127]), (5, 64, 16, 64, [(5 * i) % 40 for i in range(20)]), (1, 128, 32, 0, [4])])
def test_append(cuda, KV, D, P, N, lens, dt):
    c = cache(D + N, KV, D, P, lens, dt, spare=3 + len(lens) * (N // P + 2), M=(max(lens) + N) // P + 2)
    give_pages(c, N)
    _, kn, vn = new(N, len(lens), KV, KV, D, N, dt)
    check_append(c, kn, vn)
    assert w8.device_status() == 0


@DTYPES
def test_append_paths_and_counts(cuda, dt):
    lens = [0, 15, 16, 30, 7, 1]
    c = give_pages(cache(1, 2, 64, 16, lens, dt, spare=40, M=8), 40)
    _, kn, vn = new(2, 6, 2, 2, 64, 20, dt)
    path = torch.full((6, 9), -1, dtype=torch.int32)
    for b, p in enumerate([[0, 3, 4], [], [19], list(range(0, 18, 2)), [2, 2, 2, 1, 0, 19, 19, 5], [0, 1, 2, -1, 4, 5, 6, 7, 8]]):
        path[b, :len(p)] = torch.tensor(p, dtype=torch.int32)
    path = path.cuda()
    check_append(c, kn, vn, path=path)
    check_append(c, kn, vn, path=torch.cat([path, path], 1)[:, :9])
    count = torch.tensor([0, 20, 3, 17, 16, 1], dtype=torch.int32, device="cuda")
    check_append(c, kn, vn, count=count)
    check_append(c, kn, vn, path=path, count=count.clamp(max=9))
    check_append(c, kn, vn, path=path[:, :0])
    assert w8.device_status() == 0


@pytest.mark.parametrize("size", [1.0, 1e-30, 1e-39, 3e38])
def test_append_magnitudes(cuda, size):
    """Ties, zeros, subnormal and very large values are rounded as the definition says (bf16's range)."""
    c = give_pages(cache(1, 2, 64, 16, [0, 3], spare=9, M=4), 32)
    gen = torch.Generator(device="cuda").manual_seed(3)
    kn, vn = ((torch.randint(-256, 257, (2, 2, 32, 64), generator=gen, device="cuda") / 256.0 * size).bfloat16() for _ in range(2))
    kn[0, 0, :16] = 0
    vn[1, 1] *= 2.0 ** -100
    check_append(c, kn, vn)


@DTYPES
def test_append_values_that_are_not_finite(cuda, dt):
    """A page with one is NaN as a whole (its head's), others are as ever; the tail keeps what it is."""
    c = give_pages(cache(1, 2, 64, 16, [3, 12], dt, spare=9, M=4), 32)
    _, kn, vn = new(2, 2, 2, 2, 64, 32, dt)
    kn[0, 0, 5, 7], kn[1, 1, 20, 0], vn[0, 1, 31, 1], vn[1, 0, 2, 63] = math.inf, math.nan, -math.inf, math.nan
    check_append(c, kn, vn)
    got = run_append(c, kn, vn)
    assert bool(got["k_scale"][int(c["table"][0, 0]), 0].isnan()) and not bool(got["k_scale"][int(c["table"][0, 0]), 1].isnan())


def test_append_strides(cuda):
    c = give_pages(cache(1, 3, 128, 32, [40, 0, 31], layout="token", spare=12, M=5), 70)
    got = {n: t for n, t in c.items()}  # (in place: clones would be of another layout)
    _, kn, vn = new(2, 3, 3, 3, 128, 70, torch.bfloat16)
    kn = torch.cat([kn, kn], 3).transpose(1, 2).contiguous().transpose(1, 2)[..., :128]
    want = want_append(c, kn, vn)
    lens = w8.paged_append(c["k"], c["v"], c["k_scale"], c["v_scale"], c["k_tail"], c["v_tail"], c["table"], c["lens"], kn,
                           vn[:, :, :1].expand(-1, -1, 70, -1) if False else vn)
    for name in want:
        assert same(lens if name == "lens" else got[name], want[name]), name


@pytest.mark.parametrize("dims", [(2,), (1,), (0,), (0, 1, 2)])
def test_append_of_expanded_rows(cuda, dims):
    """New rows that stand for several tokens, heads or sequences."""
    c = give_pages(cache(1, 3, 128, 32, [40, 0, 31], spare=12, M=5), 70)
    _, kn, vn = new(2, 3, 3, 3, 128, 70, torch.bfloat16)
    for d in dims:
        kn, vn = kn.narrow(d, 0, 1).expand_as(kn), vn.narrow(d, 1, 1).expand_as(vn)
    check_append(c, kn, vn)
    path = torch.tensor([[3, 0, 69], [5, -1, 0], [1, 2, 2]], dtype=torch.int32, device="cuda")
    check_append(c, kn, vn, path=path)
    assert w8.device_status() == 0


def test_append_reports_what_is_lost(cuda):
    c = give_pages(cache(1, 1, 64, 16, [10, 10, 10, 40], spare=20, M=3), 8)
    _, kn, vn = new(2, 4, 1, 1, 64, 12, torch.bfloat16)
    before = {n: t.clone() for n, t in c.items()}

    def reported():
        with pytest.raises(w8._lib.W8InvalidArgument, match="paged cache operation"):
            w8.device_status()

    c["table"][0, 0], c["table"][1, 0] = -1, 99       # the pages of two sequences are not there
    check_append(c, kn, vn)
    reported()
    c["table"].copy_(before["table"])
    path = torch.tensor([[0, 12, 1], [99, 0, -1], [0, 1, 2], [3, -1, 0]], dtype=torch.int32, device="cuda")
    check_append(c, kn, vn, path=path)                 # new tokens that are not there: rows of zeros
    reported()
    c["lens"].copy_(torch.tensor([-1, 49, 47, 48]))    # lengths outside the table; one that it ends at
    got = run_append(c, kn, vn)
    reported()
    assert got["lens"].tolist() == [-1, 49, 48, 48]
    count = torch.tensor([-3, 99, 5, 0], dtype=torch.int32, device="cuda")
    c["lens"].copy_(before["lens"])
    got = run_append(c, kn, vn, count=count)
    reported()
    assert got["lens"].tolist() == [10, 22, 15, 40]
    assert w8.device_status() == 0


def test_append_refuses(cuda):
    c = cache(1, 1, 64, 16, [10, 3])
    _, kn, vn = new(2, 2, 1, 1, 64, 4, torch.bfloat16)
    a = [c[n] for n in ("k", "v", "k_scale", "v_scale", "k_tail", "v_tail", "table", "lens")]
    for kw, match in ((dict(lens_out=c["lens"]), "lens_out"), (dict(path=torch.zeros((2, 3), device="cuda")), "path"),
                      (dict(path=torch.zeros((1, 3), dtype=torch.int32, device="cuda")), "path"),
                      (dict(count=torch.zeros(3, dtype=torch.int32, device="cuda")), "count")):
        with pytest.raises(ValueError, match=match):
            w8.paged_append(*a, kn, vn, **kw)
    with pytest.raises(ValueError, match="expanded"):
        w8.paged_append(*a[:4], a[4][:, :, :1].expand(-1, -1, 16, -1), *a[5:], kn, vn)
    with pytest.raises(ValueError, match="k_tail"):
        w8.paged_append(*a, kn.half(), vn.half())


# ---------------------------------------------------------------- pages
def want_assign(table, lens, free, top, page, room, active, window, sink):
    table, free = [list(r) for r in table], list(free)
    M = len(table[0]) if table else 0
    rows_ = []
    for b, n in enumerate(lens):
        need = -(-(n + room) // page) if active is None or active[b] else 0
        rows_.append((need, [i < need and not (window and (i + 1) * page <= n + 1 - window and i * page >= sink) for i in range(M)]))
    for b, (need, want) in enumerate(rows_):
        for i in range(M):
            if table[b][i] >= 0 and not want[i]:
                free[top] = table[b][i]
                top += 1
                table[b][i] = -1
    have, before, ok = top, 0, []
    for b, (need, want) in enumerate(rows_):
        miss = [i for i in range(M) if want[i] and table[b][i] < 0]
        fits = need <= M
        if fits:
            before += len(miss)
        ok.append(fits and (not miss or before <= have))
        if ok[-1]:
            for i in miss:
                top -= 1
                table[b][i] = free[top]
    return table, free, top, ok


def assign_case(seed, B, M, page, room, window, sink, ended, scarce):
    r = random.Random(seed)
    pages = list(range(B * M + 5))
    r.shuffle(pages)
    lens = [r.randint(0, M * page) for _ in range(B)]
    table = []
    for n in lens:
        held = min(M, max(0, -(-n // page) + r.randint(-2, 2)))
        gone = r.randint(0, max(0, held - 1)) if window and r.random() < 0.5 else 0
        table.append([pages.pop() if gone <= i < held or (i < 1 and held) else -1 for i in range(M)])
    free = pages + [-1] * (B * M + 5 - len(pages))
    top = r.randint(0, min(len(pages), B)) if scarce else len(pages)
    active = [r.random() > 0.2 for _ in range(B)] if ended else None
    return table, lens, free, top, page, room, active, window, sink


def run_assign(table, lens, free, top, page, room, active, window, sink, width=None):
    t = torch.tensor(table, dtype=torch.int32, device="cuda").reshape(len(lens), -1)
    if width:
        t = torch.cat([t, torch.full((len(lens), width), 77, dtype=torch.int32, device="cuda")], 1)[:, :t.shape[1]]
    f, tp = torch.tensor(free, dtype=torch.int32, device="cuda"), torch.tensor([top], dtype=torch.int32, device="cuda")
    ok = w8.page_assign(t, torch.tensor(lens, dtype=torch.int32, device="cuda"), f, tp, page, room=room,
                        active=None if active is None else torch.tensor(active, device="cuda"), window=window, sink=sink)
    return t.tolist(), f.tolist(), int(tp), ok.tolist()


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("B,M,page,window,sink", [(1, 1, 16, 0, 0), (3, 7, 16, 0, 0), (8, 64, 64, 0, 0), (17, 33, 32, 100, 4),
                                                  (40, 20, 16, 50, 20), (300, 12, 128, 200, 1), (600, 41, 16, 64, 0),
                                                  (100, 200, 16, 500, 33)])
def test_page_assign(cuda, B, M, page, window, sink, seed):
    case = assign_case(seed, B, M, page, room=[1, 0, 40, 5, 16, 1000][seed], window=window, sink=sink, ended=seed % 2 == 1,
                       scarce=seed in (2, 3))
    table, free, top, ok = run_assign(*case, width=seed % 3)
    want = want_assign(*case)
    assert table == want[0] and top == want[2] and ok == want[3]
    assert free[:top] == want[1][:top]
    assert w8.device_status() == 0


def test_page_assign_many_requests(cuda):
    case = assign_case(1, 8192, 5, 16, 3, 0, 0, True, True)
    table, free, top, ok = run_assign(*case)
    want = want_assign(*case)
    assert table == want[0] and top == want[2] and ok == want[3] and free[:top] == want[1][:top]


def test_page_assign_reports(cuda):
    """Lengths out of range keep their pages; a stack that is too small, a top that is not in it."""
    def reported():
        with pytest.raises(w8._lib.W8InvalidArgument):
            w8.device_status()
        assert w8.device_status() == 0

    table, free, top, ok = run_assign([[5, 6], [7, 8], [-1, -1]], [-1, 33, 4], [1, 2, 3], 3, 16, 1, None, 0, 0)
    reported()
    assert table == [[5, 6], [7, 8], [3, -1]] and top == 2 and ok == [False, False, True]
    table, free, top, ok = run_assign([[5, 6], [7, 8]], [0, 0], [1, 2, 3], 2, 16, 0, None, 0, 0)
    reported()
    assert table == [[-1, -1], [-1, -1]] and top == 3 and free == [1, 2, 5]
    table, free, top, ok = run_assign([[-1, -1]], [20], [1, 2, 3], 9, 16, 0, None, 0, 0)
    reported()
    assert table == [[3, 2]] and top == 1


# ---------------------------------------------------------------- verification
def want_verify(logits, tokens, uniform, parent=None, draft=None, temperature=1.0, cap=0.0):
    """The walk in 64 bits, node by node."""
    B, N, V = logits.shape
    paths, taken, out = [], [], []

    def share(row, cap):
        row = row.double()
        if cap:
            row = torch.where(row == -math.inf, row, cap * torch.tanh(row / cap))
        return torch.softmax(row / temperature, 0) if bool(row.max().isfinite()) and not bool(row.isnan().any()) else None

    for b in range(B):
        up = list(range(-1, N - 1)) if parent is None else (parent if parent.dim() == 1 else parent[b]).tolist()
        path, cur, token = [0], 0, None
        while token is None:
            kids = [i for i in range(cur + 1, N) if up[i] == cur and 0 <= int(tokens[b, i]) < V]
            row = logits[b, cur].double()
            went = None
            if temperature == 0:
                if bool(row.isnan().any()) or not bool(row.max().isfinite()):
                    token = -1
                    break
                best = int(row.argmax())
                went = next((i for i in kids if int(tokens[b, i]) == best), None)
                if went is None:
                    token = best
            else:
                w = share(row, cap)
                if w is None:
                    token = -1
                    break
                q = None if draft is None else share(draft[b, cur], 0.0)
                if draft is not None and q is None:
                    kids = []
                for i in kids:
                    t = int(tokens[b, i])
                    qi = torch.zeros_like(w).index_fill_(0, torch.tensor([t], device=w.device), 1.0) if draft is None else q
                    if float(uniform[b, i]) * float(qi[t]) < float(w[t]):
                        went = i
                        break
                    rest = torch.where(qi > 0, 0.0, w) if draft is None else (w - qi).clamp(min=0)
                    if float(rest.sum()) > 1e-13:
                        w = rest / rest.sum()
                if went is None:
                    run = w.cumsum(0)
                    token = int((run > float(uniform[b, 0]) * run[-1]).int().argmax())
            if went is not None:
                path.append(went)
                cur = went
        paths.append(path + [-1] * (N - len(path)))
        taken.append(len(path))
        out.append(token)
    return paths, taken, out


def verify_case(seed, B, N, V, dt, tree, draft, temperature, pad=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    logits = (torch.randn((B, N, V), generator=gen, device="cuda") * 4).to(dt)
    near = logits.float() + torch.randn((B, N, V), generator=gen, device="cuda") * 0.7
    parent = tree_of(seed, B, N, pad)[2] if tree else None
    up = (parent if tree else torch.arange(-1, N - 1, device="cuda").expand(B, N)).long().clamp(min=0)
    tokens = torch.zeros((B, N), dtype=torch.int64, device="cuda")
    for i in range(1, N):
        row = near[torch.arange(B), up[:, i]]
        if draft:
            row = row / max(temperature, 0.01) - torch.log(-torch.log(torch.rand((B, V), generator=gen, device="cuda").clamp(1e-20, 1 - 1e-7)))
        tokens[:, i] = row.argmax(1)
    return logits, tokens, torch.rand((B, N), generator=gen, device="cuda"), parent, near.to(dt) if draft else None


def check_verify(logits, tokens, uniform, parent=None, draft=None, temperature=1.0, cap=0.0):
    path, taken, token = w8.draft_verify(logits, tokens, uniform, parent=parent, draft=draft, temperature=temperature, cap=cap)
    want = want_verify(logits, tokens, uniform, parent, draft, temperature, cap)
    assert path.tolist() == want[0] and taken.tolist() == want[1] and token.tolist() == want[2]
    return path, taken, token


@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("temperature", [0.0, 0.6, 1.0, 1.5])
@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("B,N,V,dt,tree", [
    (3, 1, 1, torch.float32, False), (4, 5, 7, torch.bfloat16, False), (5, 6, 1000, torch.float32, False),
    (6, 12, 333, torch.float16, True), (3, 16, 32000, torch.bfloat16, True), (1, 4, 262144, torch.bfloat16, False),
    (2, 3, 100003, torch.float32, True), (160, 3, 5000, torch.bfloat16, True), (7, 9, 20001, torch.float16, True)])
def test_verify(cuda, B, N, V, dt, tree, draft, temperature, cap):
    check_verify(*verify_case(N + V, B, N, V, dt, tree, draft, temperature, pad=N // 4 if tree else 0), temperature=temperature, cap=cap)
    assert w8.device_status() == 0


def test_verify_many_rejections(cuda):
    """A node with many children, nearly all of which fall: what is left shrinks again and again, the same
    token among them twice."""
    for draft in (True, False):
        logits, tokens, uniform, _, d = verify_case(5, 20, 16, 500, torch.float32, False, draft, 1.0)
        gen = torch.Generator(device="cuda").manual_seed(6)
        tokens = torch.multinomial(torch.softmax((d if draft else logits)[:, 0].float(), 1), 16, replacement=True, generator=gen)
        parent = torch.tensor([-1] + [0] * 15, dtype=torch.int32, device="cuda")
        uniform[:, 1:] = 0.5 + 0.5 * uniform[:, 1:]
        check_verify(logits, tokens, uniform, parent, d)
        tokens[:, 3] = tokens[:, 2]
        check_verify(logits, tokens, uniform, parent, d)


@pytest.mark.parametrize("V,dt,cap,temperature", [(70001, torch.float32, 0.0, 1.0), (70000, torch.bfloat16, 5.0, 0.7),
                                                  (9000, torch.float16, 0.0, 2.0), (262144, torch.bfloat16, 30.0, 1.3)])
def test_verify_many_rejections_of_wide_rows(cuda, V, dt, cap, temperature):
    """Children that fall one after the other over vocabularies of many parts, with impossible tokens in
    either model: each rejection drops some of what the one before left."""
    B, N = 6, 12
    logits, tokens, uniform, _, d = verify_case(7, B, N, V, dt, False, True, temperature)
    logits[:, :, 5::97] = -math.inf
    d[:, :, 11::89] = -math.inf
    gen = torch.Generator(device="cuda").manual_seed(8)
    tokens = torch.multinomial(torch.softmax(d[:, 0].float() / temperature, 1), N, replacement=True, generator=gen)
    parent = torch.tensor([-1] + [0] * (N - 1), dtype=torch.int32, device="cuda")
    uniform[:, 1:] = 0.6 + 0.4 * uniform[:, 1:]
    check_verify(logits, tokens, uniform, parent, d, temperature, cap)


def test_verify_uniform_ends(cuda):
    """Numbers at the ends of [0, 1): the first possible token, the last one."""
    logits, tokens, _, parent, d = verify_case(8, 6, 4, 3000, torch.float32, False, True, 1.0)
    logits[:, :, :5] = -math.inf
    logits[:, :, -3:] = -math.inf
    for u in (0.0, 1 - 2.0 ** -24):
        uniform = torch.full((6, 4), u, device="cuda")
        check_verify(logits, tokens, uniform, parent, d)
        check_verify(logits, tokens, uniform, parent, None)
        check_verify(logits, tokens, uniform, parent, None, cap=20.0)
    zero = torch.zeros((6, 1), device="cuda")
    assert w8.draft_verify(logits[:, :1], tokens[:, :1].contiguous(), zero)[2].tolist() == [5] * 6


def test_verify_impossible_and_undefined_rows(cuda):
    logits, tokens, uniform, _, d = verify_case(9, 8, 3, 600, torch.float32, False, True, 1.0)
    uniform[:, 1:] = 0  # every draft that can stand does
    logits[0, 0] = -math.inf
    logits[1, 0, 3] = math.nan
    logits[2, 0, 3] = math.inf
    logits[3, 1] = math.nan
    d[4, 0] = math.nan
    d[5, 1] = -math.inf
    logits[6, 0, int(tokens[6, 1])] = -math.inf
    for draft in (d, None):
        path, taken, token = check_verify(logits, tokens, uniform, None, draft)
        assert token.tolist()[:4] == [-1, -1, -1, -1] and taken.tolist()[3] == 2
    check_verify(logits, tokens, None, temperature=0.0)


def test_verify_equal_distributions(cuda):
    """A draft model that is the target: every draft stands, whatever the numbers."""
    logits, _, _, _, _ = verify_case(10, 50, 5, 4000, torch.bfloat16, False, True, 1.0)
    gen = torch.Generator(device="cuda").manual_seed(1)
    tokens = torch.stack([torch.zeros(50, dtype=torch.int64, device="cuda")] + [
        torch.multinomial(torch.softmax(logits[:, i].float(), 1), 1, generator=gen)[:, 0] for i in range(4)], 1)
    uniform = torch.rand((50, 5), generator=gen, device="cuda") * 0.9999
    path, taken, token = check_verify(logits, tokens, uniform, None, logits)
    assert taken.tolist() == [5] * 50


def test_verify_greedy_ties(cuda):
    """Equal largest logits: the lowest token, over the parts of a row too; -0 equals 0."""
    logits = torch.full((4, 1, 50000), -1.0, device="cuda")
    logits[0, 0, [49999, 30000, 17]] = 5.0
    logits[1, 0, [40000, 40001]] = 5.0
    logits[2, 0, 9], logits[2, 0, 44444] = -0.0, 0.0
    logits[3] = -3.0
    assert w8.draft_verify(logits, torch.zeros((4, 1), dtype=torch.int64, device="cuda"), None, temperature=0.0)[2].tolist() == [17, 40000, 9, 0]


def test_verify_strides_and_alignment(cuda):
    logits, tokens, uniform, parent, d = verify_case(11, 3, 5, 4099, torch.bfloat16, True, True, 1.0)
    wide, odd = torch.zeros((3, 7, 5000), device="cuda", dtype=torch.bfloat16), torch.zeros((3, 5, 4103), device="cuda", dtype=torch.bfloat16)
    wide[:, 1:6, 3:4102], odd[..., 1:4100] = logits, d
    for t in (1.0, 0.0):
        check_verify(wide[:, 1:6, 3:4102], tokens, uniform, parent, odd[..., 1:4100], temperature=t)
        check_verify(logits[:1].expand(3, -1, -1), tokens, uniform, parent[0], d, temperature=t)


def test_verify_chunks_of_several_turns(cuda):
    """A vocabulary of which one CTA has more than 1024 chunks of 256."""
    B, V = 149, 300001
    gen = torch.Generator(device="cuda").manual_seed(2)
    logits = torch.randn((B, 2, V), generator=gen, device="cuda") * 3
    d = logits + torch.randn((B, 2, V), generator=gen, device="cuda")
    tokens = d.argmax(2).roll(1, 1)
    uniform = torch.rand((B, 2), generator=gen, device="cuda")
    pick = [0, 1, 77, 148]
    path, taken, token = w8.draft_verify(logits, tokens, uniform, draft=d)
    want = want_verify(logits[pick], tokens[pick], uniform[pick], None, d[pick])
    assert [token.tolist()[i] for i in pick] == want[2] and [taken.tolist()[i] for i in pick] == want[1]


def test_verify_reports_tokens_out_of_range(cuda):
    logits, tokens, uniform, _, d = verify_case(12, 2, 4, 50, torch.float32, False, True, 1.0)
    tokens[0, 1], tokens[1, 1] = -1, 50
    for t in (1.0, 0.0):
        check_verify(logits, tokens, uniform, None, d, temperature=t)
        with pytest.raises(w8._lib.W8InvalidArgument, match="verification"):
            w8.device_status()
    tokens[:, 0] = 10 ** 12  # node 0's token is not looked at
    tokens[:, 1] = 0
    check_verify(logits, tokens, uniform, None, d)
    assert w8.device_status() == 0


def test_verify_keeps_the_targets_distribution(cuda):
    """Over many sequences the first token after node 0 has the target's frequencies, whatever the
    drafts (6 deviations of a count)."""
    B, V = 60000, 6
    gen = torch.Generator(device="cuda").manual_seed(4)
    row, off = torch.randn(V, generator=gen, device="cuda"), torch.randn(V, generator=gen, device="cuda")
    logits = row.expand(B, 4, V).contiguous()
    d = (row + 1.5 * off).expand(B, 4, V).contiguous()
    parent = torch.tensor([-1, 0, 0, 0], dtype=torch.int32, device="cuda")
    tokens = torch.multinomial(torch.softmax(d[:, 0], 1), 4, replacement=True, generator=gen)
    uniform = torch.rand((B, 4), generator=gen, device="cuda")
    p = torch.softmax(row.double(), 0)
    for draft in (d, None):
        path, taken, token = w8.draft_verify(logits, tokens, uniform, parent=parent, draft=draft)
        first = torch.where(taken > 1, tokens.gather(1, path[:, 1:2].long().clamp(min=0))[:, 0], token)
        if draft is None:  # (chosen without looking: the same draws would not be independent of p here)
            continue
        count = torch.bincount(first, minlength=V).double()
        assert bool(((count - B * p).abs() < 6 * (B * p * (1 - p)).sqrt()).all())


# ---------------------------------------------------------------- together
def step(c, pool, q, kn, vn, tree, depth, parent, logits, draft, tokens, uniform, N, out):
    """One step of speculative decoding over a paged cache; all on the device."""
    w8.page_assign(c["table"], c["lens"], pool["free"], pool["top"], c["k"].shape[2], room=N)
    out[0].copy_(attend(c, q, kn, vn, tree=tree, depth=depth, scale=0.09))
    path, taken, token = w8.draft_verify(logits, tokens, uniform, parent=parent, draft=draft)
    lens = w8.paged_append(c["k"], c["v"], c["k_scale"], c["v_scale"], c["k_tail"], c["v_tail"], c["table"], c["lens"], kn, vn,
                           path=path)
    c["lens"].copy_(lens)
    out[1].copy_(token)
    out[2].copy_(path)


@pytest.mark.parametrize("captured", [False, True])
def test_decoding_loop(cuda, captured):
    """Pages given out, attention, verification and append, step after step, eager and as one replayed
    graph: every step's output is the definition's over the rows so far."""
    B, H, KV, D, P, N, V, steps = 3, 8, 2, 128, 16, 6, 500, 12
    lens = [30, 0, 17]
    c = cache(1, KV, D, P, lens, spare=0, M=12)
    pages = 30
    for x in ("k", "v"):
        c[x] = torch.cat([c[x], torch.zeros((pages, KV, P, D), dtype=torch.int8, device="cuda")])
        c[x + "_scale"] = torch.cat([c[x + "_scale"], torch.zeros((pages, KV), device="cuda")])
    held = c["k"].shape[0] - pages
    free = torch.full((held + pages,), -1, dtype=torch.int32, device="cuda")
    free[:pages] = torch.arange(held, held + pages, device="cuda", dtype=torch.int32)
    pool = dict(free=free, top=torch.tensor([pages], dtype=torch.int32, device="cuda"))
    out = (torch.zeros((B, H, N, D), device="cuda", dtype=torch.bfloat16), torch.zeros(B, dtype=torch.int64, device="cuda"),
           torch.zeros((B, N), dtype=torch.int32, device="cuda"))
    tree, depth, parent = tree_of(3, B, N)
    logits, tokens, uniform, _, draft = verify_case(3, B, N, V, torch.float32, False, True, 1.0)
    q, kn, vn = new(3, B, H, KV, D, N, torch.bfloat16)
    inputs = [q, kn, vn, logits, draft, tokens, uniform]
    graph = None
    grown = 0
    for s in range(steps):
        lg, tk, un, _, dr = verify_case(100 + s, B, N, V, torch.float32, False, True, 1.0)
        for dst, src in zip(inputs, [*new(100 + s, B, H, KV, D, N, torch.bfloat16), lg, dr, tk, un]):
            dst.copy_(src)
        before = {n: t.clone() for n, t in c.items()}
        if captured and s == 1:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step(c, pool, q, kn, vn, tree, depth, parent, logits, draft, tokens, uniform, N, out)
        if graph is not None:
            graph.replay()
        else:
            step(c, pool, q, kn, vn, tree, depth, parent, logits, draft, tokens, uniform, N, out)
        kw = dict(tree=tree, depth=depth, scale=0.09)
        check_out(out[0], want_attention(before, q, kn, vn, **kw), torch.bfloat16)
        want = want_verify(logits, tokens, uniform, parent, draft)
        assert out[1].tolist() == want[2] and out[2].tolist() == want[0]
        before["table"] = c["table"].clone()  # (with the step's pages)
        after = want_append(before, kn, vn, path=out[2])
        for name in after:
            assert same(c[name], after[name]), (s, name)
        held_now = [x for x in c["table"].flatten().tolist() if x >= 0]
        assert len(set(held_now)) == len(held_now) and len(held_now) + int(pool["top"]) == held + pages
        grown += sum(want[1])
    assert grown > steps * B
    assert w8.device_status() == 0
