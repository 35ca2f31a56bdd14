"""Draft verification where the outcome hangs on a sum's last bits: certain tokens, rows at the ends of
their type, and what rejections leave.

No tolerances: a path, its length and the token are those of the definition in 64 bits, whose own
rounding moves a border by some 1e-15, or 1e-15 over what is left, where a number of the inputs lies
2^-24 from the next one.
"""
import math

import pytest
import torch

from test_paged_gpu import check_verify

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
