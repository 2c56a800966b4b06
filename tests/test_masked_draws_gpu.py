"""A token whose logit is minus infinity is never drawn, whatever the uniform number and wherever sums round."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def ops():
    from libllm_b200.csrc import ops as o
    return o


def masked_row(V, how, seed):
    """(logits with minus infinity where a token is masked, which are allowed)"""
    g = torch.Generator().manual_seed(seed)
    at = torch.arange(V)
    allowed = {"half": torch.rand(V, generator=g) < 0.5, "few": torch.rand(V, generator=g) < 0.02,
               "stretches": torch.rand((V + 99) // 100, generator=g).repeat_interleave(100)[:V] < 0.3, "first": at < 70, "last": at >= V - 3}[how]
    if not allowed.any():                                        # a row that allows nothing has no right answer
        allowed[V // 3] = True
    return torch.where(allowed, 2 * torch.randn(V, generator=g), -math.inf), allowed


@pytest.mark.parametrize("how", ["half", "few", "stretches", "first", "last"])
@pytest.mark.parametrize("V", [331, 40000])
def test_whole_vocabulary(V, how):
    """Uniform numbers all around the places where one thread's tokens end and the next one's begin, by steps of 32 bits.  A draw may lie as far from where 64 bits put
    it as the sums' roundings and the exponentials' allow: a chunk's length, the scan's twelve additions, four for the product, the exponentials and their
    arguments of up to 16, each 2^-24 of the whole: (V / 1024 + 50) 2^-24 holds them."""
    row, allowed = masked_row(V, how, V)
    weights = torch.exp(row.double() - row.max().double())
    cdf = weights.cumsum(0) / weights.sum()
    chunk = (V + 1023) // 1024
    border = cdf[torch.arange(chunk - 1, V, chunk)].float().unique()
    steps = torch.arange(-20, 21) * 2.0 ** -25
    u = torch.cat([torch.tensor([0.0, 2.0 ** -149, 2.0 ** -24, 1 - 2.0 ** -24, 1 - 2.0 ** -26]),       # the last becomes 1 in 32 bits
                   (border[:, None] * (1 + steps)).flatten(), torch.rand(4000, generator=torch.Generator().manual_seed(1))]).float().clamp_(0, 1)
    n = 4096
    rows, out = row.to(DEV).expand(n, V).contiguous(), torch.empty(n, dtype=torch.int32, device=DEV)
    drawn = []
    for part in u.split(n):
        drawn.append(ops().sample(rows[:len(part)], 1.0, 0, 1.0, part.to(DEV), out[:len(part)]).cpu())
    drawn = torch.cat(drawn).long()
    assert ((drawn >= 0) & (drawn < V)).all()
    bad = ~allowed[drawn]
    assert not bad.any(), f"{int(bad.sum())} of {len(u)} draws are of masked tokens, the first with u = {float(u[bad][0])!r}"
    tol = (V / 1024 + 50) * 2.0 ** -24
    low, high = cdf[drawn] - weights[drawn] / weights.sum(), cdf[drawn]
    assert ((u.double() >= low - tol) & (u.double() <= high + tol)).all()


@pytest.mark.parametrize("top_k,top_p", [(50, 1.0), (1024, 1.0), (50, 0.8), (0, 1.0)])
@pytest.mark.parametrize("V", [331, 20000])
def test_the_end_of_the_range(V, top_k, top_p):
    """Fewer allowed tokens than candidates, and a uniform number that is 1 in 32 bits."""
    row, allowed = masked_row(V, "last", 3)
    n = 64
    u = torch.full((n,), 1 - 2.0 ** -26, dtype=torch.float64).float()
    u[n // 2:] = torch.rand(n // 2, generator=torch.Generator().manual_seed(2))
    out = torch.empty(n, dtype=torch.int32, device=DEV)
    drawn = ops().sample(row.to(DEV).expand(n, V).contiguous(), 0.7, top_k, top_p, u.to(DEV), out).cpu().long()
    assert allowed[drawn].all(), f"{int((~allowed[drawn]).sum())} of {n} draws are of masked tokens"


@pytest.mark.parametrize("top_k,top_p", [(50, 1.0), (1024, 1.0), (50, 0.8), (1, 1.0), (0, 1.0)])
@pytest.mark.parametrize("V", [331, 20000])
def test_a_logit_that_a_penalty_took_beyond_32_bits(V, top_k, top_p):
    """A repetition far below 1 may make logits infinite: such a token stands above every other, the first of several is drawn."""
    row, allowed = masked_row(V, "half", 4)
    at = allowed.nonzero().flatten()
    row[at[7]] = row[at[20]] = 30.0                         # 30 / 1e-38 is beyond 3.4e38
    history = (~at[[7, 20]].int())[None].contiguous()
    logits = ops().adjust_logits(row[None].to(DEV), history=history.to(DEV), lengths=torch.tensor([2], dtype=torch.int32, device=DEV), repetition=1e-38)
    assert logits[0, at[7]] == math.inf and logits[0, at[20]] == math.inf and int(logits.isinf().sum()) == V - len(at) + 2
    n = 256
    u = torch.rand(n, generator=torch.Generator().manual_seed(5)).to(DEV)
    out = torch.empty(n, dtype=torch.int32, device=DEV)
    drawn = ops().sample(logits.expand(n, V).contiguous(), 0.9, top_k, top_p, u, out)
    assert (drawn == int(at[7])).all()
