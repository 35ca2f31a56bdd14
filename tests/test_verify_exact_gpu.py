"""Draft verification where the outcome hangs on a sum's last bits: certain tokens, numbers beside the
border of standing and falling, the ends of the accepted temperatures and caps, and what rejections
leave.

No tolerances: a path, its length and the token are those of the definition in 64 bits, whose own
rounding moves a border by some 1e-15, or 1e-15 over what is left, where a number of the inputs lies
2^-24 from the next one.
"""
import math

import pytest
import torch

import gemma_npu_b200 as w8
from test_paged_gpu import check_verify, want_verify

pytestmark = pytest.mark.gpu
DRAFTS = pytest.mark.parametrize("draft", [False, True], ids=["chosen", "sampled"])


def shares(row, temperature, cap=0.0):
    row = row.double()
    if cap:
        row = torch.where(row == -math.inf, row, cap * torch.tanh(row / cap))
    return torch.softmax(row / temperature, -1)


# ---------------------------------------------------------------- certain tokens
@DRAFTS
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("temperature", [1e-3, 0.1, 1.0])
def test_certain_tokens_stand(cuda, temperature, dt, draft):
    """One logit so far above the others that its probability is 1 to far more than 24 bits: its draft
    stands whatever the number, and is what is drawn."""
    B, N, V = 160, 3, 2000
    logits = torch.zeros((B, N, V), device="cuda")
    tokens = torch.zeros((B, N), dtype=torch.int64, device="cuda")
    for i in range(N):
        tokens[:, i] = (torch.arange(B, device="cuda") * 37 + i) % V
    high = 63.625 - torch.arange(B, device="cuda") / 16.0
    logits.scatter_(2, tokens.roll(-1, 1)[:, :, None], high[:, None, None].expand(B, N, 1))
    logits = logits.to(dt)
    uniform = torch.full((B, N), 1 - 2.0 ** -24, device="cuda")
    uniform[1::3] = 1 - 2.0 ** -20
    uniform[2::3] = 0.5
    path, taken, token = check_verify(logits, tokens, uniform, None, logits if draft else None, temperature)
    assert taken.tolist() == [N] * B and bool((token == tokens[:, 0]).all())


@DRAFTS
def test_rows_at_the_ends_of_the_type(cuda, draft):
    """A row may hold the type's lowest and largest values: they are numbers like others."""
    low, V = torch.finfo(torch.float32).min, 600
    logits = torch.full((8, 2, V), low, device="cuda")
    logits[1, :, 5::7] = -math.inf
    logits[2, :, 7] = 3.0
    logits[3] = -low
    logits[4, :, :9] = -low
    logits[5, :, 4] = 1e30
    logits[6] = torch.linspace(3.0e38, 3.01e38, V, device="cuda")
    logits[7, :, 3:8] = -1e33
    gen = torch.Generator(device="cuda").manual_seed(1)
    tokens = torch.randint(0, V, (8, 2), generator=gen, device="cuda")
    tokens[4, 1], tokens[5, 1], tokens[7, 1] = 3, 4, 5
    for temperature in (1.0, 1e-3, 1e3):
        for u in (0.0, 0.3, 1 - 2.0 ** -24):
            uniform = torch.full((8, 2), u, device="cuda")
            uniform[:, 1] = 0.02
            d = logits.roll(1, 0) if draft else None
            check_verify(logits, tokens, uniform, None, d, temperature)
    bf = logits.clamp(torch.finfo(torch.bfloat16).min, torch.finfo(torch.bfloat16).max).bfloat16()
    check_verify(bf, tokens, uniform, None, bf.roll(1, 0) if draft else None)


@DRAFTS
@pytest.mark.parametrize("cap", [30.0, 1e4, 1e6])
@pytest.mark.parametrize("temperature", [1e-3, 0.1, 1.0])
def test_certain_tokens_stand_under_a_cap(cuda, temperature, cap, draft):
    """The same under a softcap, whose levels fp32 has to 2^-21 of their range."""
    B, N, V = 160, 3, 2000
    logits = torch.zeros((B, N, V), device="cuda")
    tokens = (torch.arange(B, device="cuda")[:, None] * 37 + torch.arange(N, device="cuda")) % V
    high = 63.625 - torch.arange(B, device="cuda") / 16.0
    logits.scatter_(2, tokens.roll(-1, 1)[:, :, None], high[:, None, None].expand(B, N, 1))
    uniform = torch.full((B, N), 1 - 2.0 ** -24, device="cuda")
    uniform[1::3] = 1 - 2.0 ** -20
    uniform[2::3] = 0.5
    path, taken, token = check_verify(logits, tokens, uniform, None, logits if draft else None, temperature, cap)
    assert taken.tolist() == [N] * B and bool((token == tokens[:, 0]).all())


# ---------------------------------------------------------------- the accepted range
# (cap, temperature, the logits' middle, their spread): rows of a few hundred probable tokens each.
RANGE = [(0.0, 1e-3, 60.0, 4e-3), (0.0, 0.05, 60.0, 0.2), (0.0, 1.0, 20.0, 4.0), (0.0, 1e3, 0.0, 3e3), (0.0, 1.0, 6e4, 4.0),
         (30.0, 1e-3, 10.0, 4e-3), (30.0, 0.01, 25.0, 0.1), (30.0, 1.0, 20.0, 8.0), (100.0, 1.0, 0.0, 5.0),
         (1e4, 1.0, 20.0, 4.0), (1e5, 0.05, 20.0, 0.2), (1e6, 1.0, 20.0, 4.0), (1e6, 1.0, 1e6, 8.0),
         (1e-3, 1e-3, 0.0, 1e-3), (0.5, 0.02, 0.0, 0.5)]


def case_of(seed, B, N, V, middle, spread, near=0.3):
    """Target rows, rows of a draft model beside them, drafts drawn from those (of node 0's rows)."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    logits = middle + spread * torch.randn((B, N, V), generator=gen, device="cuda")
    d = logits + near * spread * torch.randn((B, N, V), generator=gen, device="cuda")
    return logits, d, gen


@pytest.mark.parametrize("cap,temperature,middle,spread", RANGE)
def test_draws_over_the_whole_range(cuda, cap, temperature, middle, spread):
    """Tokens drawn from rows without drafts."""
    logits, _, gen = case_of(7, 400, 1, 6000, middle, spread)
    uniform = torch.rand((400, 1), generator=gen, device="cuda")
    check_verify(logits, torch.zeros((400, 1), dtype=torch.int64, device="cuda"), uniform, None, None, temperature, cap)


@DRAFTS
@pytest.mark.parametrize("cap,temperature,middle,spread", RANGE)
def test_the_whole_range(cuda, cap, temperature, middle, spread, draft):
    B, N, V = 40, 5, 6000
    logits, d, gen = case_of(1, B, N, V, middle, spread)
    parent = torch.tensor([-1, 0, 0, 1, 0], dtype=torch.int32, device="cuda")
    up = torch.tensor([0, 0, 0, 1, 0], device="cuda")
    q = shares(d, temperature)[:, up]
    tokens = torch.multinomial(q.flatten(0, 1).float(), 1, generator=gen).view(B, N)
    uniform = torch.rand((B, N), generator=gen, device="cuda")
    check_verify(logits, tokens, uniform, parent, d if draft else None, temperature, cap)


def border_case(cap, temperature, middle, spread, draft):
    """A draft's number is the next one below, at or above w / q in fp32, at up to 8 steps from it."""
    B, V = 68, 6000
    logits, d, gen = case_of(2, B, 2, V, middle, spread)
    p, q = shares(logits[:, 0], temperature, cap), shares(d[:, 0], temperature)
    if draft:
        tokens = torch.multinomial(torch.where(q > p, q, 0.0).float() + 1e-30, 1, generator=gen)
        border = (p.gather(1, tokens) / q.gather(1, tokens))[:, 0]
    else:
        tokens = torch.multinomial(p.float(), 1, generator=gen)
        border = p.gather(1, tokens)[:, 0]
    steps = (torch.arange(B, device="cuda") % 17 - 8).int()
    u = (border.float().view(torch.int32) + steps).view(torch.float32).clamp(0, 1 - 2.0 ** -24)
    uniform = torch.stack([torch.rand(B, generator=gen, device="cuda"), u], 1)
    tokens = torch.cat([torch.zeros_like(tokens), tokens], 1)
    return logits, tokens, uniform, d if draft else None, u.double() / border - 1


@DRAFTS
@pytest.mark.parametrize("cap,temperature,middle,spread", RANGE)
def test_numbers_beside_the_border(cuda, cap, temperature, middle, spread, draft):
    logits, tokens, uniform, d, _ = border_case(cap, temperature, middle, spread, draft)
    path, taken, _ = check_verify(logits, tokens, uniform, None, d, temperature, cap)
    assert 10 < int((taken == 2).sum()) < 58


@DRAFTS
@pytest.mark.parametrize("cap,temperature,middle,spread", [(1e6, 0.1, -20.0, 0.4), (1e6, 1e-3, 20.0, 4e-3), (1e6, 1e-3, -3e3, 4e-3),
                                                           (1e6, 2e-3, 8e4, 0.05), (3e5, 1e-3, 1.5e4, 0.02)])
def test_numbers_beside_the_border_under_the_widest_caps(cuda, cap, temperature, middle, spread, draft):
    """Caps of up to 2^30 levels, far above the logits.  Levels (exponents of 2) of size L, up to 6e7 here, are
    rounded to 64 bits some 4 times, by 2^-53 L, on either side (the softcap's tanh, its product, the
    quotient by the temperature): each side's w is off by at most 2^-51 L ln 2, and one within 2^-50 L of its
    border may stand or fall."""
    logits, tokens, uniform, d, off = border_case(cap, temperature, middle, spread, draft)
    level = float((cap * torch.tanh(logits[:, 0].double() / cap)).abs().max()) * 1.4427 / temperature
    clear = (off.abs() > 2.0 ** -50 * level).tolist()
    path, taken, token = w8.draft_verify(logits, tokens, uniform, draft=d, temperature=temperature, cap=cap)
    want = want_verify(logits, tokens, uniform, None, d, temperature, cap)
    got = (path.tolist(), taken.tolist(), token.tolist())
    for i, on in enumerate(clear):
        assert not on or [x[i] for x in got] == [x[i] for x in want], i
    assert 10 < int((taken == 2).sum()) < 58 and sum(clear) > 50


@pytest.mark.parametrize("temperature", [0.25, 0.7, 1.0])
@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_what_a_dominant_rejected_token_leaves(cuda, cap, temperature):
    """The first chosen draft has all but 2^-21 of the probability and falls: the drafts after it are
    measured by what is left."""
    B, V = 60, 32000
    gen = torch.Generator(device="cuda").manual_seed(3)
    logits = torch.randn((B, 4, V), generator=gen, device="cuda").clamp(-4, 4) * 0.3
    first = torch.randint(0, V, (B,), generator=gen, device="cuda")
    low, up = 0.0, 100.0  # of the first draft's logit
    for _ in range(60):
        high = (low + up) / 2
        logits[:, 0].scatter_(1, first[:, None], high)
        left = 1 - float(shares(logits[0, 0], temperature, cap)[first[0]])
        low, up = (high, up) if left > 2.0 ** -21 else (low, high)
    logits[torch.arange(B), 0, (first + 1) % V] = 3.0
    w = shares(logits[:, 0], temperature, cap)
    w.scatter_(1, first[:, None], 0.0)
    w /= w.sum(1, keepdim=True)
    second = (first + 1) % V
    border = w.gather(1, second[:, None])[:, 0]
    uniform = torch.rand((B, 4), generator=gen, device="cuda")
    uniform[:, 1] = 1 - 2.0 ** -24
    uniform[:, 2] = (border * (1 + (torch.arange(B, device="cuda") % 11 - 5.5) * 1e-5)).float()
    tokens = torch.stack([torch.zeros_like(first), first, second, (first + 5) % V], 1)
    parent = torch.tensor([-1, 0, 0, 0], dtype=torch.int32, device="cuda")
    check_verify(logits, tokens, uniform, parent, None, temperature, cap)


# ---------------------------------------------------------------- what rejections leave
@pytest.mark.parametrize("near", [1e-2, 1e-4, 1e-6])
@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_rows_that_are_nearly_equal(cuda, near, cap):
    """A draft model that is nearly the target and a draft that falls all the same: the token is drawn from
    the little that is left."""
    B, V = 60, 5000
    gen = torch.Generator(device="cuda").manual_seed(4)
    logits = torch.randn((B, 2, V), generator=gen, device="cuda") * 2
    d = logits if not cap else cap * torch.tanh(logits / cap)
    d = d + near * torch.randn((B, 2, V), generator=gen, device="cuda")
    p, q = shares(logits[:, 0], 1.0, cap), shares(d[:, 0], 1.0)
    tokens = ((q - p) / q).argmax(1, keepdim=True)
    tokens = torch.cat([torch.zeros_like(tokens), tokens], 1)
    uniform = torch.rand((B, 2), generator=gen, device="cuda")
    uniform[:, 1] = 1 - 2.0 ** -24
    path, taken, _ = check_verify(logits, tokens, uniform, None, d, 1.0, cap)
    assert int((taken == 1).sum()) > (B // 2 if near > 1e-6 else 0)


@pytest.mark.parametrize("u", [0.0, 2.0 ** -24, 1 - 2.0 ** -24])
@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_the_ends_of_what_several_rejections_leave(cuda, u, cap):
    """Most of what the first rejection leaves, the front of the vocabulary among it, falls to the second
    one: the numbers at the ends find the first and last token that is left, and no other."""
    B, N, V = 96, 4, 70000
    gen = torch.Generator(device="cuda").manual_seed(5)
    logits = torch.randn((B, N, V), generator=gen, device="cuda") * 2
    flat = logits if not cap else cap * torch.tanh(logits / cap)
    d = flat - 0.05 + 0.002 * torch.rand((B, N, V), generator=gen, device="cuda")  # p / q some 1.07
    d[:, :, 30000:34000] -= 3.0
    d[:, :, 34000:60000] += 0.2
    logits[:, :, 11::97] = -math.inf
    d[:, :, 30029:34000:89] = -math.inf
    fall = torch.where(logits[:, 0, 34000:60000] == -math.inf, -math.inf, d[:, 0, 34000:60000])
    tokens = 34000 + torch.multinomial(torch.softmax(fall, 1), N, generator=gen)
    parent = torch.tensor([-1, 0, 0, 0], dtype=torch.int32, device="cuda")
    uniform = torch.full((B, N), 1 - 2.0 ** -24, device="cuda")
    uniform[:, 0] = u
    path, taken, token = check_verify(logits, tokens, uniform, parent, d, 1.0, cap)
    assert taken.tolist() == [1] * B and bool(((token >= 30000) & (token < 34000)).all())


def test_the_targets_distribution_with_chosen_drafts(cuda):
    """Chosen drafts, however they were chosen without the numbers: the first token after node 0 has the
    target's frequencies (6 deviations of a count)."""
    B, V = 60000, 6
    gen = torch.Generator(device="cuda").manual_seed(6)
    row = torch.randn(V, generator=gen, device="cuda")
    logits = row.expand(B, 4, V).contiguous()
    parent = torch.tensor([-1, 0, 0, 0], dtype=torch.int32, device="cuda")
    p = shares(row, 1.0)
    uniform = torch.rand((B, 4), generator=gen, device="cuda")
    drawn = torch.multinomial(torch.full((B, V), 1.0, device="cuda"), 4, replacement=True, generator=gen)
    best = row.argsort(descending=True)[:4].roll(1).expand(B, 4).contiguous()
    for tokens in (drawn, best):
        path, taken, token = w8.draft_verify(logits, tokens, uniform, parent=parent)
        first = torch.where(taken > 1, tokens.gather(1, path[:, 1:2].long().clamp(min=0))[:, 0], token)
        count = torch.bincount(first, minlength=V).double()
        assert bool(((count - B * p).abs() < 6 * (B * p * (1 - p)).sqrt()).all())
