"""adjust_logits against a plain 64-bit implementation."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
INF = math.inf


def ops():
    from libllm_b200.csrc import ops as o
    return o


def plain(logits, history=None, slots=None, lengths=None, repetition=1.0, presence=0.0, frequency=0.0, bias=None, allowed=None):
    """Row by row, token by token, 64-bit."""
    out = logits.double().clone()
    B, V = out.shape
    at = lambda v, b: float(v[b]) if isinstance(v, torch.Tensor) else float(v)  # noqa: E731
    for b in range(B):
        if history is not None:
            place = b if slots is None else int(slots[b])
            there = 0 <= place < history.shape[0]
            ids = history[place, :max(0, min(int(lengths[b]), history.shape[1]))].tolist() if there else []
            drawn, seen = {}, set()
            for i in ids:
                token = ~i if i < 0 else i
                if token < V:
                    seen.add(token)
                    if i >= 0:
                        drawn[token] = drawn.get(token, 0) + 1
            for v in seen:
                x = float(out[b, v])
                out[b, v] = x / at(repetition, b) if x > 0 else x * at(repetition, b)
            for v, n in drawn.items():
                out[b, v] -= at(frequency, b) * n + at(presence, b)
        if bias is not None:
            out[b] += (bias if bias.dim() == 1 else bias[b]).double()
        if allowed is not None:
            words = allowed if allowed.dim() == 1 else allowed[b]
            v = torch.arange(V)
            out[b][(words[v >> 5] >> (v & 31)) & 1 == 0] = -INF
    return out


def check(logits, **kw):
    """A logit goes through six roundings of 32 bits: two for the division by its repetition, two for the penalty, one each for taking that away and adding
    the bias.  The first two are of the logit's size, the next two of the penalty's, the last of all together: five half steps of the sum of
    what occurs on the way (the logit times its repetition, the penalty, the bias) hold them, and the plain form's narrowing."""
    o = ops()
    dev = {k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in kw.items()}
    keep = logits.to(DEV)
    before = keep.clone()
    got = o.adjust_logits(keep, **dev)
    assert torch.equal(keep.view(torch.int32), before.view(torch.int32)), "the logits were written to"
    ref = plain(logits, **kw)
    rep = kw.get("repetition", 1.0)
    rep = rep.double()[:, None] if isinstance(rep, torch.Tensor) else rep
    size = logits.double().abs() * torch.clamp(torch.as_tensor(rep, dtype=torch.float64), min=1.0)
    if kw.get("history") is not None:
        most = lambda v: float(v.abs().max()) if isinstance(v, torch.Tensor) else abs(v)  # noqa: E731
        size = size + most(kw.get("frequency", 0.0)) * kw["history"].shape[1] + most(kw.get("presence", 0.0))
    if kw.get("bias") is not None:
        size = size + kw["bias"].double().abs()
    got = got.double().cpu()
    same = (got == ref) | (got.isnan() & ref.isnan())
    far = torch.where(same, 0.0, (got - ref).abs() / (5 * 2.0 ** -24 * size + 1e-45))
    assert (far <= 1).all(), f"{int((~(far <= 1)).sum())} logits are off, by up to {float(far.nan_to_num(INF).max()):.2f} of what is allowed"
    inplace = o.adjust_logits(keep, out=keep, **dev)
    assert inplace is keep and torch.equal(keep.cpu().double().nan_to_num(7e30), got.nan_to_num(7e30))
    return got


def history_of(places, longest, V, g):
    ids = (V * torch.rand(places, longest, generator=g) ** 3).int().clamp_(max=V - 1)
    return torch.where(torch.rand(places, longest, generator=g) < 0.4, ~ids, ids).int()


def words_of(shape, V, g):
    return torch.randint(-2 ** 31, 2 ** 31, (*shape, (V + 31) // 32), generator=g).int()


@pytest.mark.parametrize("B,V,L", [(1, 1, 1), (1, 31, 5), (2, 32, 64), (3, 33, 40), (1, 1000, 3), (5, 1023, 700), (4, 8192, 100), (2, 8193, 2000),
                                   (9, 5000, 1500), (40, 2052, 333), (3, 50257, 4000), (1, 128256, 300)])
def test_everything_at_once(B, V, L):
    g = torch.Generator().manual_seed(B * V + L)
    logits = torch.randn(B, V, generator=g) * 4
    kw = dict(history=history_of(B + 2, L, V, g), slots=torch.randperm(B + 2, generator=g)[:B].int(),
              lengths=torch.randint(0, L + 1, (B,), generator=g).int(), repetition=1 + torch.rand(B, generator=g), presence=torch.rand(B, generator=g),
              frequency=0.3 * torch.rand(B, generator=g), bias=torch.randn(B, V, generator=g), allowed=words_of((B,), V, g))
    check(logits, **kw)
    for leave in ("bias", "allowed", "history"):
        check(logits, **{k: v for k, v in kw.items() if k != leave})
    check(logits, bias=kw["bias"][0], allowed=kw["allowed"][0])
    check(logits, history=kw["history"], lengths=kw["lengths"], repetition=1.3, presence=0.5, frequency=-0.25)
    check(logits, history=kw["history"], lengths=kw["lengths"], repetition=0.7)
    assert torch.equal(ops().adjust_logits(logits.to(DEV)).cpu(), logits)


def test_lengths_and_places_beyond_the_history():
    g = torch.Generator().manual_seed(1)
    V = 300
    history = history_of(4, 50, V, g)
    kw = dict(slots=torch.tensor([0, -1, 4, 3, 3, 2], dtype=torch.int32), lengths=torch.tensor([-3, 50, 50, 51, 2 ** 31 - 1, 0], dtype=torch.int32))
    check(torch.randn(6, V, generator=g), history=history, repetition=1.5, presence=1.0, frequency=0.1, **kw)


def test_ids_outside_the_vocabulary_count_for_nothing():
    history = torch.tensor([[5, 100, ~100, 2 ** 31 - 1, -2 ** 31, ~3, 99, ~99, 101]], dtype=torch.int32)
    check(torch.linspace(-3, 3, 100)[None], history=history, lengths=torch.tensor([9], dtype=torch.int32), repetition=2.0, presence=0.5, frequency=0.25)


def test_a_token_said_many_times_and_counts_of_one_history_used_twice():
    history = torch.full((2, 5000), 7, dtype=torch.int32)
    history[1, ::2] = ~8
    lengths = torch.tensor([5000, 5000, 4999], dtype=torch.int32)
    kw = dict(history=history, slots=torch.tensor([0, 1, 1], dtype=torch.int32), lengths=lengths)
    check(torch.randn(3, 40, generator=torch.Generator().manual_seed(2)), frequency=0.125, presence=0.5, repetition=1.25, **kw)


def test_infinities_and_nan():
    row = torch.tensor([INF, -INF, math.nan, 0.0, -0.0, torch.finfo(torch.float32).max, torch.finfo(torch.float32).min, 1.0])
    history = torch.arange(8).int()[None]
    allowed = torch.tensor([0b11111010], dtype=torch.int32)
    kw = dict(history=history, lengths=torch.tensor([8], dtype=torch.int32), presence=1.0, frequency=1.0)
    check(row[None], repetition=1.0, **kw)
    got = check(row[None], repetition=1.0, allowed=allowed, **kw)
    assert got[0, 0] == -INF and got[0, 2] == -INF, "a masked place is minus infinity whatever stands there"
    check(row[None], bias=torch.full((8,), -INF))


@pytest.mark.parametrize("repetition", [2.0 ** -140, 1e-39, 2.0 ** -126, 3e-38, 2.0 ** 126, 3e38, 1.0 + 2.0 ** -23, 1.0 - 2.0 ** -24])
def test_penalties_whose_reciprocal_is_no_ordinary_number(repetition):
    row = torch.tensor([1e-40, -1e-40, 2.0 ** -149, 1e-38, -1e-38, 1.0, -1.0, 3e38, -3e38, 0.0, 5e-20, -7e20])
    history = torch.arange(12).int()[None]
    got = ops().adjust_logits(row[None].to(DEV), history=history.to(DEV), lengths=torch.tensor([12], dtype=torch.int32, device=DEV),
                              repetition=torch.tensor([repetition], device=DEV))[0].cpu()
    rep = torch.tensor(repetition).double()                     # as 32 bits hold it
    want = torch.where(row > 0, row.double() / rep, row.double() * rep)
    tol = want.abs() * 2.0 ** -22 + 2.0 ** -149
    held = want.float().double()                                # infinite where 32 bits do not reach
    assert ((got.double() == held) | ((got.double() - want).abs() <= tol)).all(), (got, want)


def test_a_row_that_allows_nothing_is_still_sampled():
    o = ops()
    V = 20000
    logits = torch.randn(3, V, generator=torch.Generator().manual_seed(3)).to(DEV)
    allowed = torch.zeros(3, V // 32, dtype=torch.int32, device=DEV)
    allowed[1, 17] = 1 << 30
    got = o.adjust_logits(logits, allowed=allowed)
    assert (got[0] == -INF).all() and (got[2] == -INF).all() and int((got[1] > -INF).sum()) == 1
    out = torch.full((3,), -1, dtype=torch.int32, device=DEV)
    assert o.argmax(got, out).tolist() == [0, 17 * 32 + 30, 0]
    for top_k, top_p in ((50, 0.8), (1024, 1.0), (0, 1.0)):
        o.sample(got, 0.7, top_k, top_p, torch.tensor([0.1, 0.9, 0.5], device=DEV), out)
        drawn = out.tolist()
        assert drawn[1] == 17 * 32 + 30 and 0 <= drawn[0] < V and 0 <= drawn[2] < V


def test_rows_cut_out_of_wider_ones():
    g = torch.Generator().manual_seed(4)
    B, V, L = 6, 3001, 400
    wide, into = torch.randn(2 * B, V + 13, generator=g).to(DEV), torch.full((2 * B, V + 20), 9.0, device=DEV)
    history = history_of(2 * B, L + 9, V, g).to(DEV)
    bias, allowed = torch.randn(2 * B, V + 5, generator=g).to(DEV), words_of((2 * B,), V + 64, g).to(DEV)
    o = ops()
    for at in (0, 1, 4):
        kw = dict(history=history[::2, at:at + L], lengths=torch.full((B,), L, dtype=torch.int32, device=DEV), repetition=1.2, presence=0.4,
                  frequency=0.1, bias=bias[::2, at:at + V], allowed=allowed[::2, :(V + 31) // 32])
        x = wide[::2, at:at + V]
        got = o.adjust_logits(x, out=into[::2, at:at + V], **kw)
        assert torch.equal(got, o.adjust_logits(x.contiguous(), **{k: v.contiguous() if isinstance(v, torch.Tensor) else v for k, v in kw.items()}))
        assert (into[1::2] == 9).all() and (into[:, :at] == 9).all() and (into[:, at + V:] == 9).all()
        into.fill_(9.0)
    one = wide[:1, :V].expand(4, V)
    assert torch.equal(o.adjust_logits(one, bias=bias[0, :V]), o.adjust_logits(one.contiguous(), bias=bias[0, :V]))


def test_captured_and_replayed_with_longer_histories():
    o = ops()
    g = torch.Generator().manual_seed(5)
    logits, history = torch.randn(4, 9000, generator=g), history_of(4, 600, 9000, g)
    lengths = torch.tensor([10, 0, 100, 599], dtype=torch.int32, device=DEV)
    kw = dict(history=history.to(DEV), lengths=lengths, repetition=1.4, presence=0.3, frequency=0.2)
    x, out = logits.to(DEV), torch.empty(4, 9000, device=DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        o.adjust_logits(x, out=out, **kw)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            o.adjust_logits(x, out=out, **kw)
        lengths += 1
        graph.replay()
    s.synchronize()
    assert torch.equal(out, o.adjust_logits(x, **kw))


def test_offsets_beyond_32_bits():
    o = ops()
    g = torch.Generator().manual_seed(7)
    B, V, L, far = 2, 1000, 300, 2 ** 31 + 12
    room, ints = torch.zeros(far + 2048, device=DEV), torch.zeros(far + 2048, dtype=torch.int32, device=DEV)
    logits, history = torch.randn(B, V, generator=g).to(DEV), history_of(B, L, V, g).to(DEV)
    lengths = torch.full((B,), L, dtype=torch.int32, device=DEV)
    bias, allowed = torch.randn(B, V, generator=g).to(DEV), words_of((B,), V, g).to(DEV)
    want = o.adjust_logits(logits, history=history, lengths=lengths, repetition=1.5, frequency=0.25, bias=bias, allowed=allowed)
    x, h = room.as_strided((B, V), (far, 1)), ints.as_strided((B, L), (far, 1))
    x.copy_(logits)
    h.copy_(history)
    kw = dict(history=h, lengths=lengths, repetition=1.5, frequency=0.25, allowed=allowed)
    assert torch.equal(o.adjust_logits(x, bias=bias, **kw), want)
    o.adjust_logits(x, out=x, bias=bias, **kw)
    assert torch.equal(x, want) and int((room != 0).sum()) == int((want != 0).sum())
    b, a = room.as_strided((B, V), (far, 1)), ints.as_strided((B, allowed.shape[1]), (far, 1))
    b.copy_(bias)
    a.copy_(allowed)
    assert torch.equal(o.adjust_logits(logits, bias=b, history=history, lengths=lengths, repetition=1.5, frequency=0.25, allowed=a), want)


@pytest.mark.parametrize("repetition", [1.1, 1.2, 1.3, 1.7, 3.0, 0.7, 1.0 + 2.0 ** -23, 1.0 - 2.0 ** -24, 2.0 ** -120 * 1.1, 2.0 ** -99 * 1.3, 2.0 ** 101 * 1.9, 3e38])
@pytest.mark.parametrize("B,V", [(3, 4000), (40, 2053), (2, 8192)])
def test_a_division_by_the_repetition_is_rounded_once(repetition, B, V):
    """A token that occurs and was not drawn has its logit divided or multiplied and nothing else: the nearest number of 32 bits, which is what 64 bits
    narrow to (their quotient's own rounding, 2^-53, moves none of these across a border: a quotient of two numbers of 24 bits is no border and lies 2^-49 of itself from
    one at least).  Asked of quotients and products within the ordinary numbers, of logits whose remainders are within them too."""
    g = torch.Generator().manual_seed(V + 10 * B)
    exponent = round(math.log2(repetition) / 2)                  # logit and quotient equally far from 1
    logits = torch.randn(B, V, generator=g) * torch.exp2(torch.randint(-20, 20, (B, V), generator=g).float()) * 2.0 ** exponent
    history = (~torch.arange(V).int()).expand(B, V).contiguous()
    got = ops().adjust_logits(logits.to(DEV), history=history.to(DEV), lengths=torch.full((B,), V, dtype=torch.int32, device=DEV),
                              repetition=torch.full((B,), repetition, device=DEV)).cpu()
    by = torch.tensor(repetition).double()
    want = torch.where(logits > 0, logits.double() / by, logits.double() * by).float()
    asked = (want.abs() >= 2.0 ** -126) & want.isfinite() & (logits.abs() >= 2.0 ** -100)
    assert asked.float().mean() > 0.3
    wrong = asked & (got != want)
    assert not wrong.any(), f"{int(wrong.sum())} of {int(asked.sum())} are not the nearest"
