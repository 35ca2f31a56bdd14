"""The decoding operators (gemma_npu_b200.decode) against plain 64-bit definitions.

Tolerances.  Attention: with u = half a step of the 16-bit type (2^-8 bf16, 2^-11 fp16), the
kernel rounds each unnormalised probability once (u p_j), the output once (u |o|), and its
fp32 scores are off by at most e = (D + 4) 2^-24 scale sum|q k| + 2^-22 |x| (products summed
in fp32, one multiplication, exp2's error), which moves a probability and the sum it is
divided by by 2 e relative: |out - o| <= (u + 2 e) sum p|v| + u |o| (+ 2^-20 for the fp32
sums).  Accumulated weights: 2 e per probability and one fp32 rounding per addition.
Moved rows, integers and selections are equal bit for bit.  A selection's score: exp2's
2^-22, the argument's rounding 2^-23 max|y log2 e| (with the softcap also 2^-21 cap), one
fp32 rounding for each of the additions of a thread, and the result's rounding.
"""
import math

import pytest
import torch

import gemma_npu_b200 as w8
from gemma_npu_b200 import decode

pytestmark = pytest.mark.gpu
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def rows(gen, shape, dt, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dt)


def make(seed, B, H, KV, D, N, S, lens, dt=torch.bfloat16, layout="head"):
    """q, caches (NaN behind each length), lens, new keys and values."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    q = rows(gen, (B, H, N, D), dt, 2.0)
    if layout == "head":
        k, v = rows(gen, (B, KV, S, D), dt), rows(gen, (B, KV, S, D), dt)
    elif layout == "token":   # [B, S, KV, D] memory
        k, v = (rows(gen, (B, S, KV, D), dt).transpose(1, 2) for _ in range(2))
    else:                     # slices of a wider buffer
        k, v = (rows(gen, (B, KV + 1, S + 3, D + 24), dt)[:, 1:, 2: S + 2, 16: D + 16] for _ in range(2))
    lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    for b, n in enumerate(lens.tolist()):
        k[b, :, n:] = math.nan
        v[b, :, n:] = math.nan
    return q, k, v, lens, rows(gen, (B, KV, N, D), dt), rows(gen, (B, KV, N, D), dt)


def tree_of(seed, B, N, pad=0):
    g = torch.Generator().manual_seed(seed)
    mask, depth = torch.zeros((B, N, N), dtype=torch.bool), torch.zeros((B, N), dtype=torch.int32)
    for b in range(B):
        for i in range(N - pad):
            p = int(torch.randint(-1, i, (1,), generator=g)) if i else -1
            if p >= 0:
                mask[b, i] = mask[b, p]
                depth[b, i] = depth[b, p] + 1
            mask[b, i, i] = True
    return mask.cuda(), depth.cuda()


def want_attention(q, k, v, lens, kn, vn, tree=None, depth=None, window=0, scale=1.0):
    """(out, its tolerance without u, sum p|v|, weights of the slots, of the new tokens, their e)."""
    B, H, N, D = q.shape
    KV = k.shape[1]
    G = H // KV
    o, tol, pv = (torch.zeros((B, H, N, D), dtype=torch.float64, device="cuda") for _ in range(3))
    w = torch.zeros(k.shape[:3], dtype=torch.float64, device="cuda")
    wn = torch.zeros((B, KV, N), dtype=torch.float64, device="cuda")
    worst = 0.0
    for b, n in enumerate(lens.tolist()):
        step = torch.arange(N, device="cuda") if depth is None else (depth if depth.dim() == 1 else depth[b]).long()
        own = torch.ones((N, N), dtype=torch.bool, device="cuda").tril() if tree is None else (
            tree if tree.dim() == 2 else tree[b])
        sees = torch.cat([torch.ones((N, n), dtype=torch.bool, device="cuda"), own], 1)
        if window:
            at = torch.cat([torch.arange(n, device="cuda"), n + step])
            sees &= at[None] > (n + step)[:, None] - window
        for h in range(H):
            keys = torch.cat([k[b, h // G, :n], kn[b, h // G]]).double()
            vals = torch.cat([v[b, h // G, :n], vn[b, h // G]]).double()
            some = sees.any(0)
            keys[~some], vals[~some] = 0, 0
            x = q[b, h].double() @ keys.T * scale
            p = torch.softmax(x.masked_fill(~sees, -math.inf), 1)
            p = torch.where(sees.any(1, keepdim=True), p, 0.0)
            mag = q[b, h].double().abs() @ keys.abs().T * scale
            e = (D + 4) * 2.0 ** -24 * mag + 2.0 ** -22 * x.abs()
            e = float(torch.where(sees, e, 0.0).max()) if sees.any() else 0.0
            # each row adds only what it sees (0 * inf never happens)
            for i in range(N):
                s = sees[i]
                o[b, h, i] = p[i, s] @ vals[s]
                pv[b, h, i] = p[i, s] @ vals[s].abs()
            tol[b, h] = 2 * e * pv[b, h] + 2.0 ** -20 * pv[b, h]
            w[b, h // G, :n] += p[:, :n].sum(0)
            wn[b, h // G] += p[:, n:].sum(0)
            worst = max(worst, e)
    return o, tol, pv, w, wn, worst


def check_out(got, want, dt):
    o, tol, pv = want[:3]
    err = (got.double() - o).abs()
    bound = HALF[dt] * (pv + o.abs()) + tol + 1e-30 + (2.0 ** -24 if dt == torch.float16 else 0)
    assert bool((err <= bound).all()), float((err - bound).max())


# (B, H, KV, D, N, S, lens, window): one token; lengths around a tile and zero; groups of 1 to 8 and odd
# ones; chunks within and across tiles; windows shorter and longer than the cache.
SHAPES = [
    (1, 8, 1, 512, 1, 3700, [3658], 0),
    (1, 8, 1, 256, 1, 3700, [3658], 512),
    (6, 4, 2, 128, 1, 130, [0, 1, 63, 64, 65, 130], 0),
    (6, 4, 2, 128, 1, 130, [0, 1, 63, 64, 65, 130], 7),
    (3, 5, 1, 64, 1, 200, [200, 77, 1], 0),
    (2, 3, 3, 64, 3, 70, [70, 5], 0),
    (2, 6, 2, 128, 17, 300, [300, 129], 64),
    (1, 8, 1, 256, 70, 200, [131], 100),
    (2, 8, 8, 512, 5, 100, [64, 100], 33),
    (1, 8, 1, 512, 20, 260, [260], 128),
    (1, 2, 1, 64, 1, 1, [0], 0),
    (1, 4, 1, 128, 2, 0, [0], 0),
    (40, 32, 8, 128, 1, 100, [(7 * i) % 101 for i in range(40)], 0),
    (1, 8, 1, 256, 300, 600, [600], 512),
    (2, 16, 2, 256, 33, 500, [500, 64], 0),
    # many pieces of many rows: tiles dealt over CTAs (mma.sync), splits of row tiles (tcgen05)
    (10, 64, 4, 128, 1, 3000, [3000, 1, 700, 2999, 128, 129, 0, 2000, 64, 1500], 0),
    (10, 64, 4, 64, 1, 3000, [3000, 1, 700, 2999, 256, 257, 0, 2000, 64, 1500], 900),
    (3, 24, 2, 512, 1, 2000, [2000, 3, 1111], 0),
    (3, 8, 2, 128, 40, 4000, [4000, 2222, 31], 0),
    (1, 6, 2, 256, 50, 3000, [2900], 0),
    (300, 4, 2, 128, 1, 300, [(37 * i) % 301 for i in range(300)], 100),
    (1, 8, 1, 256, 64, 0, [0], 0),
    (1, 16, 1, 512, 3, 0, [0], 2),
    # heads of 64 of many rows: whole and odd groups, splits, windows, an empty cache
    (2, 8, 1, 64, 300, 600, [600, 0], 512),
    (1, 6, 2, 64, 50, 3000, [2900], 0),
    (9, 16, 2, 64, 40, 300, [300, 0, 1, 127, 128, 129, 255, 256, 257], 50),
    (1, 33, 1, 64, 1, 700, [650], 0),
    (1, 8, 8, 64, 130, 0, [0], 0),
    (40, 32, 1, 64, 1, 300, [(13 * i) % 301 for i in range(40)], 0),
]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("shape", SHAPES, ids=[str(i) for i in range(len(SHAPES))])
def test_chain(cuda, shape, dt):
    B, H, KV, D, N, S, lens, window = shape
    a = make(B + D + N, B, H, KV, D, N, S, lens, dt)
    got = w8.attention_tree(*a, window=window, scale=D ** -0.5)
    check_out(got, want_attention(*a, window=window, scale=D ** -0.5), dt)
    assert w8.device_status() == 0


# What few rows need more than one CTA's time for: all tiles of all sequences dealt to the resident
# CTAs.  Each head size and row tile, more than 256 sequences (which a CTA looks through in rounds),
# a window, and each of the three ways to join the pieces.
DEALT = [
    (300, 4, 1, 128, 1, 2100, [(7 * i * i) % 2101 for i in range(300)], 0),
    (300, 4, 1, 64, 1, 8000, [(31 * i * i) % 8001 for i in range(300)], 0),
    (300, 2, 1, 256, 1, 1500, [(7 * i * i) % 1501 for i in range(300)], 0),
    (300, 2, 1, 512, 1, 1000, [(7 * i * i) % 1001 for i in range(300)], 0),
    (600, 2, 1, 128, 1, 2100, [2100 - i for i in range(600)], 2000),
    (10, 64, 4, 64, 1, 20000, [20000, 1, 7000, 19999, 8000, 8193, 0, 16384, 64, 12345], 8000),
    (40, 64, 2, 128, 1, 2100, [(29 * i * i) % 2101 for i in range(40)], 0),
    (20, 64, 4, 64, 2, 3000, [(67 * i * i) % 3001 for i in range(20)], 0),
    (24, 8, 1, 256, 1, 5000, [5000 - 200 * i for i in range(24)], 0),
    (1, 32, 1, 128, 1, 3000, [2999], 0),
    (1, 16, 1, 64, 1, 9000, [9000], 0),
    (1, 11, 1, 128, 2, 3000, [3000], 2500),
]


def is_dealt(B, H, KV, D, N, S, window):
    """Few rows: only dealt tiles need a workspace when no weights are wanted."""
    assert N * H // KV <= {64: 64, 128: 32}.get(D, 16)
    return w8._lib.lib().w8_attention_tree_workspace_bytes(B, H, KV, D, S, N, window, 0) > 0


@pytest.mark.parametrize("weights", [False, True], ids=["", "weights"])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("shape", DEALT, ids=[str(i) for i in range(len(DEALT))])
def test_dealt_tiles(cuda, shape, dt, weights):
    B, H, KV, D, N, S, lens, window = shape
    assert is_dealt(B, H, KV, D, N, S, window)
    a = make(B + D + N, B, H, KV, D, N, S, lens, dt)
    prev = torch.rand((B, KV, S), device="cuda") if weights else None
    w = prev.clone() if weights else None
    got = w8.attention_tree(*a, window=window, scale=D ** -0.5, weights=w)
    want = want_attention(*a, window=window, scale=D ** -0.5)
    check_out(got[0] if weights else got, want, dt)
    if weights:
        seen = torch.arange(S, device="cuda") < a[3][:, None, None]
        exact = prev.double() + torch.where(seen, want[3], 0.0)
        rel = 2 * want[5] + (N * H // KV + 4) * 2.0 ** -24 + 2.0 ** -21
        assert ((w.double() - exact).abs() <= torch.where(seen, rel * want[3] + 2.0 ** -23 * exact, 0.0)).all()
        assert ((got[2].double() - want[4]).abs() <= rel * want[4] + 1e-30).all()
    assert w8.device_status() == 0


@pytest.mark.parametrize("shape", [(60, 4, 1, 128, 40, 1000), (60, 4, 1, 64, 40, 2000), (60, 4, 1, 256, 20, 700)], ids=str)
def test_expanded_caches_of_many_row_tiles(cuda, shape):
    """One cache for 60 sequences of several row tiles each: no TMA, rounds of pairs, tiles dealt."""
    B, H, KV, D, N, S = shape
    q, k, v, ln, kn, vn = make(D, B, H, KV, D, N, S, [S] * B)
    k, v = k[:1].expand(B, KV, S, D), v[:1].expand(B, KV, S, D)
    ln = torch.tensor([(7 * i * i) % (S + 1) for i in range(B)], dtype=torch.int32, device="cuda")
    got = w8.attention_tree(q, k, v, ln, kn, vn, scale=D ** -0.5)
    check_out(got, want_attention(q, k, v, ln, kn, vn, scale=D ** -0.5), torch.bfloat16)


# Many rows: a key axis split between clusters, of one and of two row tiles.
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("shape", [(1, 8, 1, 512, 20, 4000, [3999], 0), (1, 8, 1, 512, 40, 1500, [1500], 0), (1, 8, 1, 128, 64, 4000, [3900], 0),
                                   (2, 6, 1, 256, 50, 3000, [2900, 17], 2000)], ids=str)
def test_split_keys_of_many_rows(cuda, shape, dt):
    B, H, KV, D, N, S, lens, window = shape
    a = make(B + D + N, B, H, KV, D, N, S, lens, dt)
    w = torch.zeros((B, KV, S), device="cuda")
    got, w, _ = w8.attention_tree(*a, window=window, scale=D ** -0.5, weights=w)
    want = want_attention(*a, window=window, scale=D ** -0.5)
    check_out(got, want, dt)
    rel = 2 * want[5] + (N * H // KV + 4) * 2.0 ** -24 + 2.0 ** -21
    assert ((w.double() - want[3]).abs() <= (rel + 2.0 ** -23) * want[3]).all()


TREES = [
    (2, 8, 1, 256, 24, 300, [300, 0], 0, 0),
    (2, 8, 2, 128, 64, 150, [150, 77], 0, 5),
    (3, 4, 1, 64, 7, 64, [0, 64, 30], 0, 3),
    (1, 8, 1, 512, 9, 100, [100], 0, 2),
    (2, 8, 1, 256, 64, 400, [400, 31], 100, 4),
    (1, 4, 4, 128, 130, 90, [90], 3, 1),
    (2, 16, 2, 256, 64, 700, [700, 640], 0, 4),
    (2, 16, 2, 64, 64, 700, [700, 640], 0, 4),
    (2, 6, 2, 64, 45, 300, [300, 0], 100, 5),
    (1, 4, 4, 64, 130, 90, [90], 3, 1),
]


@pytest.mark.parametrize("layout", ["head", "token", "slice"])
@pytest.mark.parametrize("shape", TREES, ids=[str(i) for i in range(len(TREES))])
def test_tree(cuda, shape, layout):
    """Random trees with padding drafts of NaN, some with nothing to see at all."""
    B, H, KV, D, N, S, lens, window, pad = shape
    q, k, v, ln, kn, vn = make(N + D, B, H, KV, D, N, S, lens, layout=layout)
    tree, depth = tree_of(N, B, N, pad)
    if pad:
        kn[:, :, N - pad:] = math.nan
        vn[:, :, N - pad:] = math.nan
    got = w8.attention_tree(q, k, v, ln, kn, vn, tree=tree, depth=depth, window=window, scale=D ** -0.5)
    check_out(got, want_attention(q, k, v, ln, kn, vn, tree, depth, window, D ** -0.5), torch.bfloat16)
    for b, n in enumerate(lens):
        if n == 0 and pad:  # a padding draft of an empty cache sees nothing
            assert not got[b, :, N - pad:].any()


def test_shared_tree_and_strided_out(cuda):
    """One [N, N] tree and [N] depths for all sequences; q and out as token-major views."""
    B, H, KV, D, N, S = 3, 8, 2, 128, 12, 100
    _, k, v, ln, kn, vn = make(3, B, H, KV, D, N, S, [100, 50, 0])
    gen = torch.Generator(device="cuda").manual_seed(4)
    flat = rows(gen, (H, B * N, D), torch.bfloat16, 2.0)          # as qkv_norm_rope returns it
    q = flat.unflatten(1, (B, N)).transpose(0, 1)
    tree, depth = tree_of(1, 1, N)
    buf = torch.full((B, N, H, D), 7.0, dtype=torch.bfloat16, device="cuda")
    out = buf.transpose(1, 2)
    got = w8.attention_tree(q, k, v, ln, kn, vn, tree=tree[0], depth=depth[0], window=40, scale=0.1, out=out)
    assert got is out
    check_out(out, want_attention(q, k, v, ln, kn, vn, tree[0], depth[0], 40, 0.1), torch.bfloat16)


@pytest.mark.parametrize("N", [1, 11, 40])
@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_expanded_caches(cuda, D, N):
    """Beams that share one prompt's cache: k and v expanded over the batch (stride 0), q over the
    heads' batch too."""
    B, H, KV, S = 5, 4, 2, 333
    q, k, v, ln, kn, vn = make(D + N, B, H, KV, D, N, S, [333] * B)
    k, v, q = k[:1].expand(B, KV, S, D), v[:1].expand(B, KV, S, D), q[:, :1].expand(B, H, N, D)
    ln = torch.tensor([333, 300, 0, 1, 128], dtype=torch.int32, device="cuda")
    got = w8.attention_tree(q, k, v, ln, kn, vn, window=200, scale=D ** -0.5)
    check_out(got, want_attention(q, k, v, ln, kn, vn, window=200, scale=D ** -0.5), torch.bfloat16)
    assert w8.device_status() == 0


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_infinite_values_stay_with_those_who_see_them(cuda, D, dt):
    """A causal chunk whose last tokens' values are inf / NaN (a padded batch): earlier rows are
    untouched, later ones carry them."""
    B, H, KV, N, S = 2, 4, 1, 40, 90
    q, k, v, ln, kn, vn = make(D, B, H, KV, D, N, S, [90, 3], dt)
    vn[0, 0, 30, 5] = math.inf
    vn[0, 0, 33, 6] = -math.inf
    vn[0, 0, 35, 7] = math.nan
    kn[1, 0, 20] = math.nan
    got = w8.attention_tree(q, k, v, ln, kn, vn, scale=D ** -0.5)
    clean = vn.clone()
    clean[0, 0, 30, 5] = clean[0, 0, 33, 6] = clean[0, 0, 35, 7] = 0
    kc = kn.clone()
    kc[1, 0, 20] = 0
    want = want_attention(q, k, v, ln, kc, clean, scale=D ** -0.5)
    bad = torch.zeros((B, H, N, D), dtype=torch.bool, device="cuda")
    bad[0, :, 30:, 5] = bad[0, :, 33:, 6] = bad[0, :, 35:, 7] = True
    bad[1, :, 20:] = True
    check_out(torch.where(bad, want[0].to(dt), got), want, dt)
    assert (got[0, :, 30:, 5] == math.inf).all() and (got[0, :, 33:, 6] == -math.inf).all()
    assert got[0, :, 35:, 7].isnan().all() and got[1, :, 20:].isnan().all()


@pytest.mark.parametrize("D", [64, 128, 256])
def test_infinite_values_in_every_step_of_a_tile(cuda, D):
    """One non-finite value in each 16 new tokens of a warp's, few rows (mma.sync) of a tree in which
    half of the drafts see it: what follows in the same tile is computed as ever."""
    B, H, KV, N, S = 1, 1, 1, 16, 5
    q, k, v, ln, kn, vn = make(D, B, H, KV, D, 33 if D == 64 else N, S, [5])
    N = q.shape[2]
    tree = torch.ones((N, N), dtype=torch.bool, device="cuda").tril()
    tree[1::2, 0::16] = False
    tree.fill_diagonal_(True)
    clean = vn.clone()
    vn[0, 0, 0::16, 3] = math.inf
    clean[0, 0, 0::16, 3] = 0
    got = w8.attention_tree(q, k, v, ln, kn, vn, tree=tree, scale=D ** -0.5)
    want = want_attention(q, k, v, ln, kn, clean, tree, None, 0, D ** -0.5)
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[0, 0, :, 3] = tree[:, 0::16].any(1)
    check_out(torch.where(bad, want[0].to(got.dtype), got), want, torch.bfloat16)
    assert (got[bad] == math.inf).all()


def long_tail(B, H, N, D, S, large):
    """Equal keys with values 1, and keys `large` that weigh e^17.5 times as much with values 0."""
    dt = torch.float16
    q = torch.zeros((1, H, N, D), dtype=dt, device="cuda")
    q[..., 0] = 1.0
    k, v = torch.zeros((1, 1, S, D), dtype=dt, device="cuda"), torch.ones((1, 1, S, D), dtype=dt, device="cuda")
    k[0, 0, large, 0], v[0, 0, large] = 17.5, 0.0
    kn, vn = torch.zeros((1, 1, N, D), dtype=dt, device="cuda"), torch.ones((1, 1, N, D), dtype=dt, device="cuda")
    lens = torch.full((B,), S, dtype=torch.int32, device="cuda")
    one = q, k, v, lens[:1], kn, vn
    return one, [x.expand(B, *x.shape[1:]) for x in (q, k, v)] + [lens] + [x.expand(B, *x.shape[1:]) for x in (kn, vn)]


# Each of fp16's probabilities may be half a step of its least one off (2^-25) where the sum is at
# least 2^7: 2^-32 a key, whose values are at most 1 here.  Lost altogether they would sum to some
# S e^-17.5 / (number of large keys): 1.5e-3 and 4.7e-5 against bounds of 1.4e-5 and 7.4e-6.
@pytest.mark.parametrize("case", [(1, 70, 64, 60000), (1, 40, 128, 60000), (1, 20, 256, 60000), (1, 20, 512, 60000),
                                  (1200, 1, 64, 30000), (1200, 1, 128, 30000)], ids=str)
def test_fp16_keeps_a_long_tail_of_small_weights(cuda, case):
    """tcgen05 (one large key), and the warps of mma.sync CTAs that hold a whole sequence each (a
    large key in every 16 of their first ones)."""
    B, N, D, S = case
    one, all_of = long_tail(B, 8 if B == 1 else 1, N, D, S, [100] if B == 1 else list(range(0, 256, 16)))
    o, tol, pv = want_attention(*one)[:3]
    err = (w8.attention_tree(*all_of).double() - o).abs()
    assert bool((err <= HALF[torch.float16] * (pv + o) + tol + 2.0 ** -24 + 2.0 ** -32 * (S + N)).all()), float(err.max())


@pytest.mark.parametrize("D,N", [(64, 1), (128, 40), (256, 2), (512, 20)])
def test_fp16_accumulated_weights_of_a_long_tail(cuda, D, N):
    one, _ = long_tail(1, 8, N, D, 9000, [100])
    w = torch.zeros((1, 1, 9000), device="cuda")
    _, wo, dw = w8.attention_tree(*one, weights=w)
    want = want_attention(*one)
    rel = 2 * want[5] + (8 * N + 4) * 2.0 ** -24 + 2.0 ** -21
    assert ((wo.double() - want[3]).abs() <= rel * want[3]).all() and ((dw.double() - want[4]).abs() <= rel * want[4]).all()


@pytest.mark.parametrize("N", [1, 40])
@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_slots_before_the_window_may_hold_anything(cuda, D, N):
    """NaN in the committed slots that no token's window reaches, inside the first tile read."""
    B, H, KV, S, W = 2, 4, 1, 700, 100
    q, k, v, ln, kn, vn = make(D + N, B, H, KV, D, N, S, [700, 333])
    want = want_attention(q, k, v, ln, kn, vn, window=W, scale=D ** -0.5)
    for b, n in enumerate([700, 333]):
        k[b, :, :n - W + 1] = math.nan
        v[b, :, :n - W + 1] = math.nan
    check_out(w8.attention_tree(q, k, v, ln, kn, vn, window=W, scale=D ** -0.5), want, torch.bfloat16)


WEIGHTS = [
    (1, 8, 1, 256, 1, 3000, [2900], 0, False),
    (4, 8, 2, 128, 1, 300, [300, 0, 64, 131], 0, False),
    (2, 4, 1, 64, 5, 100, [100, 40], 30, False),
    (2, 8, 1, 256, 40, 200, [200, 0], 0, True),
    (1, 8, 1, 512, 10, 150, [149], 60, True),
    (24, 32, 8, 128, 1, 500, [20 * i + 7 for i in range(24)], 0, False),
    # many rows
    (2, 16, 2, 64, 121, 14, [14, 3], 0, True),
    (1, 8, 1, 128, 90, 1100, [1030], 300, False),
    (2, 17, 1, 64, 1, 600, [600, 129], 0, False),
    (2, 8, 1, 256, 35, 260, [255, 0], 64, True),
]


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("shape", WEIGHTS, ids=[str(i) for i in range(len(WEIGHTS))])
def test_weights(cuda, shape, in_place):
    B, H, KV, D, N, S, lens, window, tree = shape
    a = make(S, B, H, KV, D, N, S, lens)
    tr, dp = tree_of(2, B, N) if tree else (None, None)
    gen = torch.Generator(device="cuda").manual_seed(9)
    prev = torch.rand((B, KV, S), generator=gen, device="cuda")
    w = prev.clone()
    to = None if in_place else torch.full_like(prev, -3.0)
    o, wo, dw = w8.attention_tree(*a, tree=tr, depth=dp, window=window, scale=D ** -0.5, weights=w, weights_out=to)
    want = want_attention(*a, tr, dp, window, D ** -0.5)
    check_out(o, want, torch.bfloat16)
    assert wo is (w if in_place else to)
    G, e = H // KV, want[5]
    rel = 2 * e + (G * N + 4) * 2.0 ** -24 + 2.0 ** -21
    for b, n in enumerate(lens):
        exact = prev[b, :, :n].double() + want[3][b, :, :n]
        assert ((wo[b, :, :n].double() - exact).abs() <= rel * want[3][b, :, :n] + 2.0 ** -23 * exact).all()
        assert torch.equal(wo[b, :, n:], (prev if in_place else torch.full_like(prev, -3.0))[b, :, n:])
    assert ((dw.double() - want[4]).abs() <= rel * want[4] + 1e-30).all()
    if not in_place:
        assert torch.equal(w, prev)


def test_weights_of_no_new_tokens(cuda):
    """N = 0 adds nothing: the weights of the committed slots still go to weights_out."""
    S, lens = 2600, [2600, 5, 0]
    q, k, v, ln, kn, vn = make(1, 3, 4, 2, 64, 3, S, lens)
    wide = torch.rand((3, 2, S + 9), device="cuda")
    w, to = wide[..., 2:S + 2], torch.full((3, 2, S), -3.0, device="cuda")
    empty = q[:, :, :0], k, v, ln, kn[:, :, :0], vn[:, :, :0]
    o, wo, dw = w8.attention_tree(*empty, weights=w, weights_out=to)
    assert o.shape == (3, 4, 0, 64) and wo is to and dw.shape == (3, 2, 0)
    for b, n in enumerate(lens):
        assert torch.equal(to[b, :, :n], w[b, :, :n]) and (to[b, :, n:] == -3).all()
    before = wide.clone()
    assert w8.attention_tree(*empty, weights=w)[1] is w and torch.equal(wide, before)
    assert w8.device_status() == 0


@pytest.mark.parametrize("N", [1, 3, 60])
def test_same_bits_every_time(cuda, N):
    a = make(1, 2, 8, 1, 256, N, 3000, [3000, 1234])
    w = torch.rand((2, 1, 3000), device="cuda")
    first = w8.attention_tree(*a, scale=0.06, weights=w, weights_out=torch.zeros_like(w))
    for _ in range(3):
        for x, y in zip(first, w8.attention_tree(*a, scale=0.06, weights=w, weights_out=torch.zeros_like(w))):
            assert torch.equal(x, y)


def test_a_length_outside_the_cache_is_reported(cuda):
    q, k, v, ln, kn, vn = make(1, 2, 4, 1, 64, 1, 80, [80, 80])
    over = torch.tensor([81, -1], dtype=torch.int32, device="cuda")
    got = w8.attention_tree(q, k, v, over, kn, vn, scale=0.1)
    with pytest.raises(w8._lib.W8InvalidArgument, match="outside its range"):
        w8.device_status()
    assert w8.device_status() == 0
    inside = torch.tensor([80, 0], dtype=torch.int32, device="cuda")
    assert torch.equal(got, w8.attention_tree(q, k, v, inside, kn, vn, scale=0.1))


def test_offsets_past_32_bits(cuda):
    """A cache of more than 2^31 elements: its last slots."""
    D, S = 512, (1 << 22) + 100
    k = torch.zeros((1, 1, S, D), dtype=torch.bfloat16, device="cuda")
    v = torch.zeros((1, 1, S, D), dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(1)
    n, W = S - 3, 70
    k[0, 0, n - W:n], v[0, 0, n - W:n] = rows(gen, (W, D), torch.bfloat16), rows(gen, (W, D), torch.bfloat16)
    q, kn, vn = (rows(gen, s, torch.bfloat16) for s in ((1, 8, 2, D), (1, 1, 2, D), (1, 1, 2, D)))
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    got = w8.attention_tree(q, k, v, lens, kn, vn, window=W, scale=0.05)
    short = torch.tensor([W], dtype=torch.int32, device="cuda")
    want = want_attention(q, k[:, :, n - W:n], v[:, :, n - W:n], short, kn, vn, window=W, scale=0.05)
    check_out(got, want, torch.bfloat16)
    new = w8.cache_append(k, v, kn, vn, lens)
    assert new.item() == n + 2 and torch.equal(k[0, 0, n:n + 2], kn[0, 0]) and torch.equal(v[0, 0, n:n + 2], vn[0, 0])
    assert not k[0, 0, n + 2:].any() and not k[0, 0, :100].any()


# ---------------------------------------------------------------- append
APPENDS = [(1, 1, 64, 10, 1, None), (3, 2, 128, 100, 40, None), (4, 2, 256, 50, 9, [[0, 2, 5], [8, -1, 3], [-1, 1, 1], [1, 4, 4]]),
           (2, 5, 512, 30, 20, [list(range(20)), [19 - i for i in range(17)] + [-1, -1, 0]]), (2, 1, 64, 8, 3, [[], []])]


@pytest.mark.parametrize("layout", ["head", "token", "slice"])
@pytest.mark.parametrize("shape", APPENDS, ids=[str(i) for i in range(len(APPENDS))])
def test_append(cuda, shape, layout):
    B, KV, D, S, N, path = shape
    lens = [(11 * b) % (S - N + 1) for b in range(B)]
    _, k, v, ln, kn, vn = make(N, B, KV, KV, D, N, S, lens, layout=layout)
    gen = torch.Generator(device="cuda").manual_seed(2)
    w, dw = torch.rand((B, KV, S), generator=gen, device="cuda"), torch.rand((B, KV, N), generator=gen, device="cuda")
    pos = torch.full((B, KV, S), -1, dtype=torch.int32, device="cuda")
    seen = torch.tensor([1000 + b for b in range(B)], dtype=torch.int32, device="cuda")
    k0, v0, w0 = k.clone(), v.clone(), w.clone()
    p = None if path is None else torch.tensor(path, dtype=torch.int32, device="cuda").reshape(B, -1)
    out = w8.cache_append(k, v, kn, vn, ln, path=p, weights=w, draft_weights=dw, positions=pos, seen=seen)
    for b in range(B):
        take = list(range(N)) if path is None else path[b]
        take = take[:take.index(-1)] if -1 in take else take
        n, m = lens[b], lens[b] + len(take)
        assert out[b].item() == m
        k0[b, :, n:m], v0[b, :, n:m], w0[b, :, n:m] = kn[b][:, take], vn[b][:, take], dw[b][:, take]
        assert pos[b, :, n:m].tolist() == [[1000 + b + j for j in range(len(take))]] * KV
        assert (pos[b, :, :n] == -1).all() and (pos[b, :, m:] == -1).all()
    for got, want in ((k, k0), (v, v0), (w, w0)):
        assert torch.equal(got.nan_to_num(5.0), want.nan_to_num(5.0))
    assert w8.device_status() == 0


def test_append_skips_what_is_out_of_range(cuda):
    """A full cache, a draft index that is none and a bad length: skipped and reported."""
    _, k, v, _, kn, vn = make(5, 3, 1, 1, 64, 4, 10, [10, 10, 10])
    k0 = k.clone()
    ln = torch.tensor([8, 2, -5], dtype=torch.int32, device="cuda")
    path = torch.tensor([[0, 1, 2], [0, 4, 1], [0, 1, 2]], dtype=torch.int32, device="cuda")
    out = w8.cache_append(k, v, kn, vn, ln, path=path)
    k0[0, :, 8:10] = kn[0, :, :2]
    k0[1, :, 2], k0[1, :, 4] = kn[1, :, 0], kn[1, :, 1]
    assert torch.equal(k, k0) and out.tolist() == [10, 5, -5]
    with pytest.raises(w8._lib.W8InvalidArgument):
        w8.device_status()
    assert w8.device_status() == 0


def test_append_refuses_to_write_lengths_over_what_it_reads(cuda):
    _, k, v, ln, kn, vn = make(5, 2, 2, 2, 64, 3, 20, [4, 9])
    pos = torch.zeros((2, 2, 20), dtype=torch.int32, device="cuda")
    buf = torch.zeros(4, dtype=torch.int32, device="cuda")
    for kw in (dict(positions=pos, seen=buf[:2], lens_out=buf[:2]), dict(positions=pos, seen=buf[:2], lens_out=buf[1:3]),
               dict(path=buf[:2].view(2, 1), lens_out=buf[1:3])):
        with pytest.raises(w8._lib.W8InvalidArgument, match="lens_out"):
            w8.cache_append(k, v, kn, vn, ln, **kw)
    with pytest.raises(w8._lib.W8InvalidArgument, match="lens_out"):
        w8.cache_append(k, v, kn, vn, buf[:2], lens_out=buf[1:3])
    assert not buf.any() and w8.device_status() == 0


@pytest.mark.parametrize("dt", [torch.int8, torch.float32, torch.float16])
def test_append_moves_any_rows(cuda, dt):
    k, v = (torch.zeros((2, 3, 9, 16), dtype=dt, device="cuda") for _ in range(2))
    new = torch.randint(-100, 100, (2, 3, 2, 16), device="cuda").to(dt)
    ln = torch.tensor([0, 7], dtype=torch.int32, device="cuda")
    w8.cache_append(k, v, new, new + 1, ln, weights=(w := torch.ones((2, 3, 9), device="cuda")))
    for b, n in enumerate([0, 7]):
        assert torch.equal(k[b, :, n:n + 2], new[b]) and torch.equal(v[b, :, n:n + 2], new[b] + 1)
        assert not w[b, :, n:n + 2].any()


# ---------------------------------------------------------------- evict
def want_evict(k, v, w, pos, lens, budget, sink, recent):
    k, v, wo, po = k.clone(), v.clone(), torch.zeros_like(w), torch.full_like(pos, -1)
    for b, n in enumerate(lens):
        for h in range(k.shape[1]):
            ww, pp = w[b, h, :n].tolist(), pos[b, h, :n].tolist()
            src = list(range(min(n, budget)))
            if n > budget:
                top = max(pp)
                safe = [p < sink or p > top - recent for p in pp]
                val = [-math.inf if x != x else x for x in ww]
                kept = set(sorted(range(n), key=lambda s: (not safe[s], -val[s], s))[:budget])
                holes = [s for s in range(budget) if s not in kept]
                for d, s in zip(holes, sorted(s for s in kept if s >= budget)):
                    src[d] = s
            k[b, h, :len(src)], v[b, h, :len(src)] = k[b, h, src], v[b, h, src]
            wo[b, h, :len(src)], po[b, h, :len(src)] = w[b, h, src], pos[b, h, src]
    return k, v, wo, po, [min(n, budget) for n in lens]


EVICTS = [(1, 1, 64, 10, [10], 4, 0, 0), (3, 2, 128, 700, [700, 100, 0], 100, 4, 20), (2, 1, 256, 3000, [3000, 2999], 1024, 4, 128),
          (2, 2, 64, 2100, [2049, 1025], 1, 0, 1), (1, 1, 128, 1500, [1500], 1499, 2, 1000), (1, 2, 64, 50, [50], 50, 0, 0),
          (1, 1, 64, 40, [33], 60, 0, 0), (1, 1, 512, 33000, [33000], 5000, 8, 100), (2, 1, 64, 5000, [5000, 4097], 4096, 0, 4096)]


# Rows above 8192 slots, few and many, up to and beyond what a cluster's registers hold.
EVICTS += [(1, 1, 64, 8193, [8193], 1000, 4, 100), (1, 3, 64, 16500, [16385], 12000, 0, 11000), (9, 1, 64, 9000, [9000, 0, 500, 8999, 1, 501, 499, 4096, 8193], 500, 4, 20),
           (30, 1, 64, 8200, [8200 - 250 * i for i in range(30)], 700, 4, 20), (40, 2, 64, 9000, [9000 - 200 * i for i in range(40)], 700, 4, 20),
           (2, 1, 64, 32769, [32769, 20000], 20000, 4, 20), (1, 1, 64, 70000, [69990], 3000, 4, 100), (1, 1, 64, 131072, [131072], 65536, 1, 1),
           (1, 1, 64, 131100, [131100], 4000, 1, 1), (1, 1, 64, 100000, [100000], 99999, 50000, 49999), (1, 1, 64, 40000, [3000], 3000, 0, 0)]


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("kind", ["random", "ties", "odd"])
@pytest.mark.parametrize("shape", EVICTS, ids=[str(i) for i in range(len(EVICTS))])
def test_evict(cuda, shape, kind, in_place):
    B, KV, D, S, lens, budget, sink, recent = shape
    gen = torch.Generator(device="cuda").manual_seed(S)
    k, v = rows(gen, (B, KV, S, D), torch.bfloat16), rows(gen, (B, KV, S, D), torch.bfloat16)
    w = torch.exp(3 * torch.randn((B, KV, S), generator=gen, device="cuda"))
    if kind == "ties":
        w = torch.randint(0, 3, (B, KV, S), generator=gen, device="cuda").float()
    if kind == "odd":
        special = torch.tensor([math.nan, math.inf, -math.inf, 0.0, -0.0, -1.5, 1e-45, 3e38], device="cuda")
        w = special[torch.randint(0, 8, (B, KV, S), generator=gen, device="cuda")]
    pos = torch.argsort(torch.rand((B, KV, S), generator=gen, device="cuda"), dim=2).int() * 3
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    want = want_evict(k, v, w, pos, lens, budget, sink, recent)
    wo, po = (w, pos) if in_place else (None, None)
    got = w8.cache_evict(k, v, w, pos, ln, budget, sink=sink, recent=recent, weights_out=wo, positions_out=po)
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    assert torch.equal(got[0].nan_to_num(-7.0, posinf=9.0, neginf=-9.0), want[2].nan_to_num(-7.0, posinf=9.0, neginf=-9.0))
    assert torch.equal(got[1], want[3]) and got[2].tolist() == want[4]
    assert w8.device_status() == 0


# ---------------------------------------------------------------- beam search
def want_select(logits, scores, finished, pad, n, cap, order):
    B, K, V = logits.shape
    y = logits.double()
    if cap > 0:
        y = torch.where(y == -math.inf, y, cap * torch.tanh(y / cap))
    total = scores.double()[:, :, None] + (y - torch.logsumexp(y, 2, keepdim=True))
    if finished is not None:
        total[finished] = -math.inf
        total[finished, pad] = scores.double()[finished]
    total = torch.where(torch.isfinite(total), total, -math.inf)
    out = []
    for b in range(B):
        flat = sorted(range(K * V), key=lambda i: (-total[b].flatten()[i].item(), i)) if K * V <= 512 else \
            torch.sort(total[b].flatten(), descending=True, stable=True)[1][:n].tolist()
        picks = [(total[b].flatten()[i].item(), i // V, i % V) for i in flat[:n]]
        if order == "slot":
            taken, free, placed = set(), [s for s in range(K) if s not in {p[1] for p in picks}], [None] * K
            for p in picks:
                s = p[1] if p[1] not in taken else free.pop(0)
                taken.add(s)
                placed[s] = p
            picks = placed
        out.append(picks)
    return out


def check_select(got, want, y_max, V, cap):
    s, beam, token = got
    tol = 2.0 ** -22 + 2.0 ** -23 * y_max * 1.45 * 2 + (V / 256 + 40) * 2.0 ** -24 + 2.0 ** -21 * cap * 1.45
    for b, picks in enumerate(want):
        assert beam[b].tolist() == [p[1] for p in picks]
        assert token[b].tolist() == [p[2] for p in picks]
        for x, p in zip(s[b].tolist(), picks):
            assert x == p[0] or abs(x - p[0]) <= tol + 2.0 ** -24 * abs(p[0])


SELECTS = [(1, 4, 262144, 4, 0.0, "score"), (2, 3, 50001, 6, 30.0, "score"), (3, 8, 4097, 8, 0.0, "slot"), (1, 1, 7, 7, 0.0, "score"),
           (2, 32, 300, 64, 30.0, "score"), (2, 32, 9000, 32, 0.0, "slot"), (4, 5, 3, 10, 0.0, "score"), (1, 2, 200000, 1, 30.0, "score"),
           (7, 16, 1000, 16, 30.0, "slot"), (20, 8, 30000, 16, 0.0, "score"), (1, 16, 1, 16, 0.0, "score")]


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("shape", SELECTS, ids=[str(i) for i in range(len(SELECTS))])
def test_select(cuda, shape, dt):
    B, K, V, n, cap, order = shape
    gen = torch.Generator(device="cuda").manual_seed(V + n)
    logits = rows(gen, (B, K, V), dt, 4.0)
    scores = torch.randn((B, K), generator=gen, device="cuda") * 2 - 9
    got = w8.beam_select(logits, scores, n=n, cap=cap, order=order)
    check_select(got, want_select(logits, scores, None, 0, n, cap, order), 24.0, V, cap)


@pytest.mark.parametrize("order", ["score", "slot"])
@pytest.mark.parametrize("V", [64, 5000, 70000])
def test_select_ties(cuda, V, order):
    """Beams with the same logits and scores, logits of few values, one beam all equal."""
    B, K = 2, 6
    gen = torch.Generator(device="cuda").manual_seed(V)
    row = torch.randint(-2, 3, (B, 1, V), generator=gen, device="cuda").float()
    logits = row.repeat(1, K, 1)
    logits[:, 3] = 0.5
    scores = torch.full((B, K), -2.0, device="cuda")
    scores[1, 4] = -1.0
    got = w8.beam_select(logits, scores, order=order)
    check_select(got, want_select(logits, scores, None, 0, K, 0.0, order), 4.0, V, 0.0)


@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("n", [4, 8])
def test_select_impossible(cuda, n, cap):
    """-inf logits and scores, finished beams over rows of NaN, beams without a finite sum."""
    B, K, V, pad = 5, 4, 300, 7
    gen = torch.Generator(device="cuda").manual_seed(1)
    logits = rows(gen, (B, K, V), torch.float32, 3.0)
    scores = torch.randn((B, K), generator=gen, device="cuda") - 5
    finished = torch.zeros((B, K), dtype=torch.bool, device="cuda")
    scores[0, 1:] = -math.inf                     # the first step
    logits[1, :, 3:] = -math.inf                  # three possible tokens each
    finished[2, 1:] = True
    logits[2, 1:] = math.nan                      # a finished beam's logits are not read
    finished[3] = True                            # fewer continuations than asked for
    scores[3, 2] = -math.inf
    logits[4, 0, 5] = math.nan                    # no finite sum
    logits[4, 1] = -math.inf
    scores[4, 2] = math.nan
    want = want_select(logits, scores, finished, pad, n, cap, "score")
    got = w8.beam_select(logits, scores, finished=finished, pad=pad, n=n, cap=cap)
    check_select(got, want, 16.0, V, cap)


@pytest.mark.parametrize("kind", ["saturated", "rounded"])
@pytest.mark.parametrize("n", [1, 5, 24])
def test_select_orders_a_beam_by_its_logits(cuda, n, kind):
    """Different logits whose scores are equal in 64 bits, by a saturated softcap or by rounding:
    the logits decide within a beam, the lower beam between beams."""
    B, K, V, cap = 2, 3, 500, 30.0 if kind == "saturated" else 0.0
    gen = torch.Generator(device="cuda").manual_seed(n)
    few = torch.randint(0, 40, (B, K, V), generator=gen, device="cuda").float()
    logits = 700 + 5 * few if kind == "saturated" else 1e-20 * few
    logits[:, 2, 100:] = -5.0
    scores = torch.tensor([[-1.0, -1.0, -1.0], [-2.0, -1.0, -1.5]], device="cuda")
    got = w8.beam_select(logits, scores, n=n, cap=cap)
    for b in range(B):
        every = []
        for k in range(K):
            x = logits[b, k].double()
            y = cap * torch.tanh(x / cap) if cap else x
            total = (scores[b, k].double() + (y - torch.logsumexp(y, 0))).tolist()
            order = sorted(range(V), key=lambda t: (-x[t].item(), t))[:n]
            assert len({total[t] for t in order}) == 1 and (n < 24 or len({x[t].item() for t in order}) > 1)
            every += [(-total[t], k, i, t) for i, t in enumerate(order)]
        every = sorted(every)[:n]
        assert got[1][b].tolist() == [e[1] for e in every] and got[2][b].tolist() == [e[3] for e in every]
        assert all(abs(s + e[0]) <= 1e-4 for s, e in zip(got[0][b].tolist(), every))


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("cap", [1e-30, 1e-4, 5e-3, 0.5, 999.0, 1001.0, 1e4, 1e6, 1e30])
def test_select_scores_under_any_cap(cuda, cap, dt):
    """Caps far below and far above the logits; whole segments of zeros.  A softcapped logit is off by
    at most 2^-21 of the smaller of the cap and the logit."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    B, K, V, n = 2, 3, 9000, 4
    logits = rows(gen, (B, K, V), dt, 4.0)
    logits[:, :, 160:320] = 0
    scores = torch.randn((B, K), generator=gen, device="cuda") - 5
    got = w8.beam_select(logits, scores, n=n, cap=cap)[0].double()
    total = scores.double()[:, :, None] + torch.log_softmax(cap * torch.tanh(logits.double() / cap), 2)
    want = torch.topk(total.reshape(B, -1), n).values
    tol = 2.0 ** -22 + 2.0 ** -23 * 24 * 1.45 * 2 + (V / 256 + 40) * 2.0 ** -24 + 2.0 ** -21 * min(cap, 24.0) * 1.45
    assert ((got - want).abs() <= tol + 2.0 ** -24 * want.abs()).all(), (got - want).abs().max()


@pytest.mark.parametrize("cap", [math.nan, math.inf, 1e-46, 1e-31, 1e31, 1e300])
def test_select_refuses_caps_it_cannot_scale(cuda, cap):
    logits, scores = torch.zeros((1, 2, 9), device="cuda"), torch.zeros((1, 2), device="cuda")
    with pytest.raises(ValueError, match="cap must be"):
        w8.beam_select(logits, scores, cap=cap)
    assert w8.beam_select(logits, scores, cap=-cap if cap == cap else -1.0)[0].isfinite().all()  # not positive: none


@pytest.mark.parametrize("order", ["", "scores", "\udc80", "sl\0ot", "slot\0", b"slot", None, 0])
def test_select_refuses_other_orders(cuda, order):
    """Text that no UTF-8 encodes among them."""
    with pytest.raises(ValueError, match="order must be"):
        w8.beam_select(torch.zeros((1, 2, 9), device="cuda"), torch.zeros((1, 2), device="cuda"), order=order)


@pytest.mark.parametrize("kind", ["rising", "falling", "equal", "first"])
def test_select_orders_that_fill_the_candidates(cuda, kind):
    """Ascending logits pass every threshold; equal ones tie on all of them."""
    V = 40000
    base = torch.arange(V, device="cuda", dtype=torch.float32) / 4096
    row = {"rising": base, "falling": -base, "equal": torch.zeros(V, device="cuda"),
           "first": torch.where(base == 0, 1.0, -1.0)}[kind]
    logits = row.repeat(1, 2, 1).contiguous()
    scores = torch.tensor([[-1.0, -1.5]], device="cuda")
    got = w8.beam_select(logits, scores, n=64)
    check_select(got, want_select(logits, scores, None, 0, 64, 0.0, "score"), 16.0, V, 0.0)


def test_select_strided_and_unaligned_rows(cuda):
    gen = torch.Generator(device="cuda").manual_seed(3)
    wide = rows(gen, (3, 5, 1003), torch.bfloat16, 4.0)
    logits = wide[:, 1:4, 1:1002]
    scores = torch.randn((3, 3), generator=gen, device="cuda")
    got = w8.beam_select(logits, scores)
    check_select(got, want_select(logits, scores, None, 0, 3, 0.0, "score"), 24.0, 1001, 0.0)


@pytest.mark.parametrize("n", [2, 64])
@pytest.mark.parametrize("found", [64, 100, 121, 125, 126, 127, 128, 129, 200])
def test_select_segments_that_nearly_fill_the_candidates(cuda, found, n):
    """The best value in `found` segments of 16 logits (their first one, or all of them): as many
    candidates as are held at once, one segment less or more, while the collection adds to their number."""
    B, V = 6, 4096
    gen = torch.Generator(device="cuda").manual_seed(found)
    logits = -torch.rand((B, 1, V), generator=gen, device="cuda") - 1
    for b in range(B):
        at = torch.randperm(V // 16, generator=gen, device="cuda")[:found]
        if b % 2:
            logits[b].view(-1, 16)[at] = 2.0
        else:
            logits[b].view(-1, 16)[at, 0] = 2.0
    scores = torch.linspace(-1, -1.5, B, device="cuda")[:, None].contiguous()
    for _ in range(20):
        got = w8.beam_select(logits, scores, n=n)
    check_select(got, want_select(logits, scores, None, 0, n, 0.0, "score"), 2.0, V, 0.0)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("n", [4, 64])
@pytest.mark.parametrize("kind", ["random", "late", "ties"])
def test_select_in_several_collections(cuda, kind, n, dt):
    """Chunks of more than 24 tiles, whose later collections start from the candidates of the first:
    random logits, the best in the later tiles, and few values (ties across the collections)."""
    B, K, V, tile = 50, 8, 262144, 4096
    ws = w8._lib.lib().w8_beam_select_workspace_bytes(B, K, V, n)
    chunks = ws // (B * K * (n * 8 + 8))
    assert V // tile // chunks > 24
    gen = torch.Generator(device="cuda").manual_seed(n)
    logits = rows(gen, (B, K, V), torch.float32, 4.0)
    if kind == "late":
        logits += 3.0 * ((torch.arange(V, device="cuda") // tile) % (V // tile // chunks) >= 24)
    if kind == "ties":
        logits = logits.round().clamp(max=11.0)
    logits = logits.to(dt)
    scores = torch.randn((B, K), generator=gen, device="cuda") - 9
    got = w8.beam_select(logits, scores, n=n)
    check_select(got, want_select(logits, scores, None, 0, n, 0.0, "score"), 28.0, V, 0.0)


REORDERS = [(1, 4, 1, 256, 100, 3), (2, 3, 2, 64, 33, 1), (3, 8, 2, 128, 64, 5), (1, 32, 1, 64, 17, 2), (2, 16, 3, 64, 50, 70), (4, 1, 1, 64, 5, 1)]


@pytest.mark.parametrize("index", [torch.int64, torch.int32])
@pytest.mark.parametrize("ragged", [True, False])
@pytest.mark.parametrize("shape", REORDERS, ids=[str(i) for i in range(len(REORDERS))])
def test_reorder(cuda, shape, ragged, index):
    """Any map of beams, swaps and cycles included, in place; rows behind the length stay."""
    B, K, heads, D, S, count = shape
    gen = torch.Generator(device="cuda").manual_seed(K)
    caches = [rows(gen, (B * K, S, heads, D), torch.bfloat16).transpose(1, 2) for _ in range(count)]
    beam = torch.randint(0, K, (B, K), generator=gen, device="cuda")
    beam[0] = torch.arange(K, device="cuda").roll(1)
    lens = torch.randint(0, S + 1, (B * K,), generator=gen, device="cuda").int() if ragged else None
    want = [c.clone() for c in caches]
    for r in range(B * K):
        src = r - r % K + int(beam[r // K, r % K])
        n = int(lens[src]) if ragged else S
        for c, y in zip(caches, want):
            y[r, :, :n] = c[src, :, :n]
    assert w8.cache_reorder(caches, beam.to(index), lens=lens) is caches
    for c, y in zip(caches, want):
        assert torch.equal(c, y)
    assert w8.device_status() == 0


def test_reorder_takes_one_layout_whatever_its_idle_strides(cuda):
    """Dimensions of one element may have any stride; any other difference of layout is refused."""
    x, y = torch.randn((4, 1, 8, 16), device="cuda"), torch.randn((4, 8, 1, 16), device="cuda").transpose(1, 2)
    assert x.stride() != y.stride()
    beam, src = torch.tensor([[1, 0], [0, 0]], device="cuda"), [1, 0, 2, 2]
    want = [x[src], y[src]]
    w8.cache_reorder([x, y], beam)
    assert torch.equal(x, want[0]) and torch.equal(y, want[1])
    for other in (torch.randn((4, 1, 9, 16), device="cuda")[:, :, :8], torch.randn((8, 4, 1, 16), device="cuda").permute(1, 2, 0, 3)):
        with pytest.raises(ValueError, match="one shape, layout"):
            w8.cache_reorder([x, other], beam)


def test_reorder_bad_parents_are_reported(cuda):
    x = torch.randn((4, 1, 8, 16), device="cuda")
    want = x.clone()
    want[3] = x[2]
    w8.cache_reorder(x, torch.tensor([[9, -1, 2, 2]], device="cuda"))
    assert torch.equal(x, want)
    with pytest.raises(w8._lib.W8InvalidArgument):
        w8.device_status()


# ---------------------------------------------------------------- streams, graphs, refusals
def test_captured_graphs_share_nothing(cuda):
    """Two graphs captured on one stream, replayed at the same time on two others with new
    inputs, give what eager calls give."""
    def step(s):
        o, w, dw = w8.attention_tree(*s["a"], scale=0.06, weights=s["w"], weights_out=s["wo"])
        picks = w8.beam_select(s["logits"], s["scores"])
        ev = w8.cache_evict(s["k"], s["v"], s["w"], s["pos"], s["a"][3], 500, sink=2, recent=50)
        return (o, w, dw) + picks + ev + (s["k"],)

    def state(seed):
        a = make(seed, 2, 8, 1, 256, 1, 2000, [2000, 1000])
        gen = torch.Generator(device="cuda").manual_seed(seed)
        return dict(a=a, w=torch.rand((2, 1, 2000), generator=gen, device="cuda"), wo=torch.zeros((2, 1, 2000), device="cuda"),
                    logits=rows(gen, (2, 4, 30000), torch.float32, 4.0), scores=torch.zeros((2, 4), device="cuda"),
                    k=rows(gen, (2, 1, 2000, 64), torch.bfloat16), v=rows(gen, (2, 1, 2000, 64), torch.bfloat16),
                    pos=torch.arange(2000, device="cuda", dtype=torch.int32).repeat(2, 1, 1))

    states = [state(1), state(2)]
    wants = [[t.clone() for t in step(s)] for s in states]
    graphs, outs = [], []
    torch.cuda.synchronize()
    for s in states:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(s))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for out, want in zip(outs, wants):
        for x, y in zip(out, want):
            assert torch.equal(x, y)


def test_side_stream(cuda):
    """On another stream the call is ordered on that stream."""
    st = torch.cuda.Stream()
    a = make(1, 2, 8, 2, 128, 1, 600, [600, 300])
    want = w8.attention_tree(*a, scale=0.1)
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        q = a[0] * 1  # made on the side stream
        got = w8.attention_tree(q, *a[1:], scale=0.1)
    st.synchronize()
    assert torch.equal(got, want)


def test_refusals(cuda):
    q, k, v, ln, kn, vn = make(1, 2, 4, 2, 64, 3, 20, [20, 5])
    tree, depth = tree_of(1, 2, 3)
    ok = dict(scale=0.1)
    bad = [
        ((q.float(), k, v, ln, kn, vn), ok), ((q, k.half(), v, ln, kn, vn), ok), ((q, k, v, ln.long(), kn, vn), ok),
        ((q[:, :3], k, v, ln, kn, vn), ok), ((q, k, v[:, :, :9], ln, kn, vn), ok), ((q, k, v, ln, kn[:, :, :2], vn), ok),
        ((q, k, v, ln[:1], kn, vn), ok), ((q, k, v, ln.cpu(), kn, vn), ok), ((q.cpu(), k, v, ln, kn, vn), ok),
        ((q, k, v, ln, kn, vn), dict(tree=tree.int())), ((q, k, v, ln, kn, vn), dict(tree=tree[:, :2])),
        ((q, k, v, ln, kn, vn), dict(tree=tree, window=4)), ((q, k, v, ln, kn, vn), dict(depth=depth.long())),
        ((q, k, v, ln, kn, vn), dict(window=-1)), ((q, k, v, ln, kn, vn), dict(out=torch.empty_like(q)[:, :, :2])),
        ((q, k, v, ln, kn, vn), dict(out=q.new_empty((1, 1, 3, 64)).expand(2, 4, 3, 64))),
        ((q, k, v, ln, kn, vn), dict(weights_out=torch.zeros((2, 2, 20), device="cuda"))),
        ((q, k, v, ln, kn, vn), dict(weights=torch.zeros((2, 2, 19), device="cuda"))),
        ((q.transpose(2, 3), k, v, ln, kn, vn), ok), ((q[..., :48], k[..., :48], v[..., :48], ln, kn[..., :48], vn[..., :48]), ok),
    ]
    for args, kw in bad:
        with pytest.raises((ValueError, w8.W8Error)):
            w8.attention_tree(*args, **kw)
    wide = torch.zeros((2, 4, 3, 67), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(w8._lib.W8AlignmentError):
        w8.attention_tree(wide[..., 1:65], k, v, ln, kn, vn)
    w = torch.zeros((2, 2, 20), device="cuda")
    pos = torch.zeros((2, 2, 20), dtype=torch.int32, device="cuda")
    for kw in (dict(budget=0), dict(budget=5, sink=3, recent=3), dict(budget=5, sink=-1), dict(budget=5, lens_out=ln)):
        with pytest.raises((ValueError, w8.W8Error)):
            w8.cache_evict(k, v, w, pos, ln, **kw)
    for kw in (dict(path=ln), dict(draft_weights=w), dict(positions=pos), dict(lens_out=ln), dict(path=tree[:, 0])):
        with pytest.raises((ValueError, w8.W8Error)):
            w8.cache_append(k, v, kn, vn, ln, **kw)
    with pytest.raises((ValueError, w8.W8Error)):
        w8.cache_append(k[:, :1].expand(2, 2, 20, 64), v, kn, vn, ln)
    logits, scores = torch.zeros((2, 3, 10), device="cuda"), torch.zeros((2, 3), device="cuda")
    for kw in (dict(n=31), dict(n=0), dict(n=65), dict(n=4, order="slot"), dict(order="best"), dict(pad=10), dict(pad=-1),
               dict(finished=scores), dict(finished=torch.zeros((2, 2), dtype=torch.bool, device="cuda"))):
        with pytest.raises((ValueError, w8.W8Error)):
            w8.beam_select(logits, scores, **kw)
    with pytest.raises((ValueError, w8.W8Error)):
        w8.beam_select(torch.zeros((1, 33, 10), device="cuda"), torch.zeros((1, 33), device="cuda"))
    x, beam = torch.zeros((6, 1, 4, 64), device="cuda"), torch.zeros((2, 3), dtype=torch.int64, device="cuda")
    for args in ((x[:5], beam), (x, beam.float()), ([x, x], beam), ([x, x[:, :, :2]], beam), (x, beam.cpu())):
        with pytest.raises((ValueError, w8.W8Error)):
            w8.cache_reorder(*args)
    with pytest.raises((ValueError, w8.W8Error)):
        w8.cache_reorder(torch.zeros((6, 1, 4, 6), device="cuda"), beam)
    assert w8.device_status() == 0


def test_empty_calls(cuda):
    q, k, v, ln, kn, vn = make(1, 2, 4, 2, 64, 3, 20, [20, 5])
    assert w8.attention_tree(q[:0], k[:0], v[:0], ln[:0], kn[:0], vn[:0]).shape == (0, 4, 3, 64)
    assert w8.attention_tree(q[:, :, :0], k, v, ln, kn[:, :, :0], vn[:, :, :0]).shape == (2, 4, 0, 64)
    assert w8.cache_append(k, v, kn[:, :, :0], vn[:, :, :0], ln).tolist() == [20, 5]
    assert w8.beam_select(torch.zeros((0, 2, 9), device="cuda"), torch.zeros((0, 2), device="cuda"))[0].shape == (0, 2)
    assert w8.cache_reorder([], torch.zeros((1, 2), dtype=torch.int64, device="cuda")) == []


def test_beam_search_with_eviction(cuda):
    """A run of them together: beams decode over their caches, the head's logits are selected
    from, the states follow, the caches are cut by weight; every step's attention and
    selection is checked against histories kept as lists."""
    B, K, H, KV, D, S, V, budget = 2, 4, 8, 2, 64, 48, 600, 24
    gen = torch.Generator(device="cuda").manual_seed(7)
    emb = rows(gen, (V, 128), torch.bfloat16)
    proj = rows(gen, (128, (H + 2 * KV) * D), torch.bfloat16, 128 ** -0.5)
    back = rows(gen, (H * D, 128), torch.bfloat16, (H * D) ** -0.5)
    head_q, head_s = w8.quant_rows(rows(gen, (V, 128), torch.bfloat16))
    head_s = head_s.to(torch.bfloat16)
    R = B * K
    k, v = (torch.full((R, KV, S, D), math.nan, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    lens = torch.zeros(R, dtype=torch.int32, device="cuda")
    weights = torch.zeros((R, KV, S), device="cuda")
    pos = torch.full((R, KV, S), -1, dtype=torch.int32, device="cuda")
    scores = torch.full((B, K), -math.inf, device="cuda")
    scores[:, 0] = 0
    token = torch.zeros((B, K), dtype=torch.int64, device="cuda")
    hist = [[{} for _ in range(KV)] for _ in range(R)]  # per state and head: position -> [k row, v row, weight]
    for step in range(40):
        y = (emb[token.flatten()] @ proj).view(R, 1, H + 2 * KV, D).transpose(1, 2)
        q, kn, vn = y[:, :H], y[:, H:H + KV], y[:, H + KV:]
        o, _, dw = w8.attention_tree(q, k, v, lens, kn, vn, scale=D ** -0.5, weights=weights)
        for r in range(R):
            for h in range(KV):
                items = sorted(hist[r][h].items())
                keys = torch.stack([x[0] for _, x in items] + [kn[r, h, 0]]).double()
                vals = torch.stack([x[1] for _, x in items] + [vn[r, h, 0]]).double()
                qs = q[r, h * (H // KV):(h + 1) * (H // KV), 0].double()
                p = torch.softmax(qs @ keys.T * D ** -0.5, 1)
                err = (o[r, h * (H // KV):(h + 1) * (H // KV), 0].double() - p @ vals).abs()
                assert (err <= 2.0 ** -8 * (p @ vals.abs() + (p @ vals).abs()) + 2.0 ** -12).all()
                for (at, x), add in zip(items, p.sum(0).tolist()):
                    x[2] += add
                hist[r][h][step] = [kn[r, h, 0].clone(), vn[r, h, 0].clone(), p.sum(0)[-1].item()]
        seen = torch.full((R,), step, dtype=torch.int32, device="cuda")
        lens = w8.cache_append(k, v, kn, vn, lens, weights=weights, draft_weights=dw, positions=pos, seen=seen)
        logits = w8.int8_linear(o[:, :, 0].reshape(R, H * D) @ back, head_q, head_s).view(B, K, V)
        got = w8.beam_select(logits, scores, cap=30.0, order="slot")
        check_select(got, want_select(logits, scores, None, 0, K, 30.0, "slot"), 30.0, V, 30.0)
        scores, beam, token = got
        w8.cache_reorder([k, v], beam, lens=lens)
        src = (beam + torch.arange(B, device="cuda")[:, None] * K).flatten()
        weights, pos, lens = weights[src].contiguous(), pos[src].contiguous(), lens[src].contiguous()
        hist = [[{a: list(x) for a, x in hist[s][h].items()} for h in range(KV)] for s in src.tolist()]
        weights, pos, lens = w8.cache_evict(k, v, weights, pos, lens, budget, sink=2, recent=6)
        for r in range(R):
            n = int(lens[r])
            assert n == min(step + 1, budget)
            for h in range(KV):
                kept = pos[r, h, :n].tolist()
                left = [a for a in hist[r][h] if a not in kept]
                assert len(set(kept)) == n and set(range(min(2, step + 1))) <= set(kept)
                floor = min((hist[r][h][a][2] for a in kept if 2 <= a <= step - 6), default=math.inf)
                assert all(hist[r][h][a][2] <= floor * (1 + 1e-5) for a in left)
                for a in left:
                    del hist[r][h][a]
    assert w8.device_status() == 0
