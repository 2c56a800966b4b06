"""The output end of a step in the engine: the output matrix in four bits, penalties, biases and masks before the draw, in every way that a
token can come to a sequence."""
import numpy as np
import pytest
import torch

import plain_four_bits as Q
import plain_llama as P
from helpers import TINY, model_folder, plain_weights, rms_err, tokens_for

pytestmark = pytest.mark.gpu


def engine(name="C", dtype="float32", **kw):
    from libllm_b200.engine import Engine
    kw.setdefault("max_tokens", 2048)
    return Engine.from_folder(model_folder(name), dtype=dtype, **kw)


class Sequence:
    """What a sequence holds, told apart as the penalties tell it: (token, drawn)."""

    def __init__(self, slot):
        self.slot, self.tokens, self.fresh = slot, [], None

    def bring(self, tokens):
        for i, t in enumerate(tokens):
            self.tokens.append((t, i == 0 and self.fresh == t))
            self.fresh = None
        return self


def adjusted(logits, seq, s):
    """One row of logits as SamplingParams asks for it, 64-bit, token by token."""
    x = logits.astype(np.float64).copy()
    drawn = {}
    for t, d in seq.tokens:
        drawn[t] = drawn.get(t, 0) + bool(d)
    for t, n in drawn.items():
        x[t] = x[t] / s.repetition_penalty if x[t] > 0 else x[t] * s.repetition_penalty
        if n:
            x[t] -= s.frequency_penalty * n + s.presence_penalty
    for t, v in s.logit_bias:
        x[t] += v
    return x


def is_best(token, x, what):
    """The token is the largest of x, or so near it that 32-bit rounding (five of them, of numbers up to the largest) may have put it first."""
    slack = 5 * 2.0 ** -24 * np.abs(x[np.isfinite(x)]).max()
    assert x[token] >= x.max() - 2 * slack, f"{what}: token {token} has {x[token]}, the best is {x.max()}"


def greedy(**kw):
    from libllm_b200.engine import SamplingParams
    return SamplingParams(temperature=0.0, top_k=1, top_p=1.0, **kw)


def run(e, seqs, tokens, s, fed=None, allowed=None, want=None):
    """One step; checks every drawn token and notes it."""
    from libllm_b200.engine import StepItem
    items = [StepItem(q.slot, t if fed is None or fed[i] is None else [0], [len(t) - 1] if want is None or want[i] else [],
                      None if fed is None else fed[i]) for i, (q, t) in enumerate(zip(seqs, tokens))]
    logits, drawn = e.step(items, s, None, True, allowed)
    for q, t in zip(seqs, tokens):
        q.bring(t)
    rows = [q for i, q in enumerate(seqs) if want is None or want[i]]
    for r, q in enumerate(rows):
        x = adjusted(logits[r], q, s)
        if allowed is not None:
            x[~allowed[r]] = -np.inf
        is_best(int(drawn[r]), x, f"slot {q.slot} at {len(q.tokens)}")
        q.fresh = int(drawn[r])
    return [int(t) for t in drawn]


# ---------------------------------------------------------------- penalties
@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_penalties_in_steps(dtype, graphs):
    e = engine(dtype=dtype, track_history=True, use_graphs=graphs, max_slots=8)
    s = greedy(repetition_penalty=1.3, presence_penalty=0.02, frequency_penalty=0.03)
    a, b = Sequence(e.open_sequence()), Sequence(e.open_sequence())
    drawn = run(e, [a, b], [tokens_for("C", 40, 1), tokens_for("C", 3, 2)], s)
    for i in range(12):                                      # drawn tokens brought back by their ids
        drawn = run(e, [a, b], [[drawn[0]], [drawn[1]]], s)
    drawn = run(e, [b], [[drawn[1]]], s)                     # one alone, then a turn that nobody drew, then both again
    run(e, [a], [tokens_for("C", 9, 3)], s)
    last = run(e, [a, b], [[5], [drawn[0]]], s)
    run(e, [b, a], [[last[1]], [last[0]]], s)
    assert sum(d for _, d in a.tokens) >= 12 and sum(d for _, d in b.tokens) >= 13
    # a slot that another sequence had
    e.close_sequence(a.slot)
    c = Sequence(e.open_sequence())
    assert c.slot == a.slot
    first = run(e, [c], [[t for t, _ in a.tokens[:45]]], s)
    run(e, [c], [first], s)


@pytest.mark.parametrize("graphs", [True, False])
def test_drawn_tokens_that_stay_on_the_device(graphs):
    from libllm_b200.engine import StepItem
    e = engine(track_history=True, use_graphs=graphs)
    s = greedy(repetition_penalty=1.2, presence_penalty=0.05, frequency_penalty=0.05)
    prompts = [tokens_for("C", 20, 4), tokens_for("C", 7, 5)]
    seqs = [Sequence(e.open_sequence()) for _ in prompts]
    pending = e.step_tokens([StepItem(q.slot, p, [len(p) - 1]) for q, p in zip(seqs, prompts)], s)
    got = [pending.result()]
    for _ in range(10):
        pending = e.step_tokens([StepItem(q.slot, [0], [0], row) for row, q in enumerate(seqs)], s)
        got.append(pending.result())
    other = engine(track_history=True, use_graphs=graphs)     # the same by ids, with the logits read and checked
    seqs = [Sequence(other.open_sequence()) for _ in prompts]
    want = [run(other, seqs, prompts, s)]
    for _ in range(10):
        want.append(run(other, seqs, [[t] for t in want[-1]], s))
    assert got == want


def test_a_prompt_cut_into_pieces():
    whole = engine(track_history=True)
    cut = engine(track_history=True, max_step_tokens=16)
    s = greedy(repetition_penalty=1.5, presence_penalty=0.1, frequency_penalty=0.1)
    for n in (15, 16, 17, 50):
        toks = [t % 40 for t in tokens_for("C", n, n)]
        for e in (whole, cut):
            q = Sequence(e.open_sequence())
            t = run(e, [q], [toks], s)
            for _ in range(3):
                t = run(e, [q], [t], s)
            e.close_sequence(q.slot)


def test_what_a_sequence_that_wants_nothing_draws_is_nobodys():
    e = engine(track_history=True)
    s = greedy(repetition_penalty=1.3, presence_penalty=0.5, frequency_penalty=0.5)
    a, b = Sequence(e.open_sequence()), Sequence(e.open_sequence())
    drawn = run(e, [a, b], [tokens_for("C", 10, 6), tokens_for("C", 11, 7)], s)
    for i in range(4):
        # b wants nothing in every other step: what comes next for it counts as brought, also where it is the token that was computed for it
        want = [True, i % 2 == 0]
        drawn_now = run(e, [a, b], [[drawn[0]], [drawn[1]]], s, want=want)
        drawn = [drawn_now[0], drawn_now[1] if want[1] else drawn[1]]


def test_generate_and_complete_with_penalties():
    from libllm_b200 import Model
    from libllm_b200.engine import SamplingParams
    m = Model(model_folder("C"), dtype="float32", max_tokens=2048, track_history=True)
    prompts = [tokens_for("C", 12, 8), tokens_for("C", 5, 9), tokens_for("C", 30, 10)]
    kw = dict(temperature=0.0, repetition_penalty=1.4, presence_penalty=0.1, frequency_penalty=0.2, logit_bias={3: 0.05, 100: -0.2})
    got = m.generate(prompts, 12, stop_token_ids=[], **kw)
    e = engine(track_history=True)
    s = SamplingParams(top_k=1, top_p=1.0, **kw)
    for p, tokens in zip(prompts, got):
        q = Sequence(e.open_sequence())
        t = run(e, [q], [p], s)
        mine = list(t)
        for _ in range(11):
            t = run(e, [q], [t], s)
            mine += t
        assert mine == tokens
        e.close_sequence(q.slot)
        assert [c.token for c in m.complete(p, max_new_tokens=12, **kw)] == tokens
    # without penalties the same engine draws as one that tracks nothing
    assert m.generate(prompts, 12, temperature=0.0, stop_token_ids=[]) == \
        Model(model_folder("C"), dtype="float32", max_tokens=2048).generate(prompts, 12, temperature=0.0, stop_token_ids=[])


# ---------------------------------------------------------------- biases and masks
@pytest.mark.parametrize("graphs", [True, False])
def test_biases_change_from_step_to_step(graphs):
    e = engine(use_graphs=graphs)
    q = Sequence(e.open_sequence())
    t = run(e, [q], [tokens_for("C", 6, 11)], greedy(logit_bias={17: 50.0}))
    assert t == [17]
    for bias, drawn in (({17: 50.0}, 17), ({3: 40.0, 17: 30.0}, 3), ([(330, 99.0)], 330), ({}, None), ({0: 60.0}, 0), ({17: 50.0}, 17)):
        t = run(e, [q], [t], greedy(logit_bias=bias))
        assert drawn is None or t == [drawn]


@pytest.mark.parametrize("graphs", [True, False])
def test_masks(graphs):
    e = engine(use_graphs=graphs, track_history=True)
    V, rng = e.vocab, np.random.default_rng(5)
    s = greedy(repetition_penalty=1.2)
    seqs = [Sequence(e.open_sequence()) for _ in range(3)]
    drawn = run(e, seqs, [tokens_for("C", n, n) for n in (4, 9, 2)], s, allowed=rng.random((3, V)) < 0.1)
    for i in range(4):
        allowed = rng.random((3, V)) < 0.05
        drawn = run(e, seqs, [[t] for t in drawn], s, allowed=allowed)
        assert all(allowed[r, t] for r, t in enumerate(drawn))
    allowed = np.zeros((2, V), dtype=bool)
    allowed[0, V - 1] = allowed[1, 0] = True
    got = run(e, seqs, [[t] for t in drawn], s, allowed=allowed, want=[True, False, True])
    assert got == [V - 1, 0]
    run(e, seqs, [[V - 1], [drawn[1]], [0]], s)              # and none again


def test_masks_as_bits_and_a_mask_that_allows_nothing():
    from libllm_b200.engine import StepItem
    e = engine()
    V = e.vocab
    words = np.zeros((1, (V + 31) // 32), dtype=np.uint32)
    words[0, 5] = 1 << 31
    slot = e.open_sequence()
    assert e.step([StepItem(slot, [1, 2, 3], [2])], greedy(), None, True, words)[1].tolist() == [5 * 32 + 31]
    assert e.step([StepItem(slot, [4], [0])], greedy(), None, True, words.view(np.int32))[1].tolist() == [5 * 32 + 31]
    for s in (greedy(), None):
        if s is None:
            from libllm_b200.engine import SamplingParams
            s = SamplingParams()
        for tokens in ([5], [6, 7]):
            t = e.step([StepItem(slot, tokens, [len(tokens) - 1])], s, [0.5], True, np.zeros((1, V), dtype=bool))[1]
            assert 0 <= int(t[0]) < V


def test_the_logits_that_come_back_are_the_models_own():
    from libllm_b200.engine import StepItem
    e, plain = engine(track_history=True), engine()
    s = greedy(repetition_penalty=2.0, presence_penalty=1.0, frequency_penalty=1.0, logit_bias={1: 5.0})
    toks = tokens_for("C", 30, 12)
    a, b = e.open_sequence(), plain.open_sequence()
    assert np.array_equal(e.step([StepItem(a, toks, [29])], s)[0], plain.step([StepItem(b, toks, [29])]))
    for t in toks[:4]:
        assert np.array_equal(e.step([StepItem(a, [t], [0])], s, None, True, np.ones((1, e.vocab), dtype=bool))[0], plain.step([StepItem(b, [t], [0])]))


# ---------------------------------------------------------------- refusals
def test_refusals():
    from libllm_b200.engine import Engine, StepItem
    from libllm_b200.errors import InvalidArgError
    e = engine()
    tracked = engine(track_history=True)
    slot, other = e.open_sequence(), tracked.open_sequence()
    ones = np.ones((1, e.vocab), dtype=bool)
    for call in (
            lambda: e.step([StepItem(slot, [1], [0])], greedy(repetition_penalty=1.1)),
            lambda: e.generate([[1, 2]], 2, greedy(presence_penalty=0.1)),
            lambda: list(e.complete([1, 2], greedy(frequency_penalty=0.1), 2)),
            lambda: tracked.step([StepItem(other, [1, 2], [0])], greedy(repetition_penalty=1.1)),
            lambda: tracked.step([StepItem(other, [1, 2], [0, 1])], greedy(repetition_penalty=1.1)),
            lambda: tracked.step([StepItem(other, [1], [0])], greedy(repetition_penalty=0.0)),
            lambda: tracked.step([StepItem(other, [1], [0])], greedy(repetition_penalty=-2.0)),
            lambda: tracked.step([StepItem(other, [1], [0])], greedy(repetition_penalty=float("nan"))),
            lambda: tracked.step([StepItem(other, [1], [0])], greedy(repetition_penalty=1e300)),
            lambda: tracked.step([StepItem(other, [1], [0])], greedy(presence_penalty=float("inf"))),
            lambda: e.step([StepItem(slot, [1], [0])], greedy(logit_bias={e.vocab: 1.0})),
            lambda: e.step([StepItem(slot, [1], [0])], greedy(logit_bias={-1: 1.0})),
            lambda: e.step([StepItem(slot, [1], [0])], greedy(logit_bias=[(1, 1.0), (1, 2.0)])),
            lambda: e.step([StepItem(slot, [1], [0])], greedy(logit_bias={1: float("nan")})),
            lambda: e.step([StepItem(slot, [1], [0])], None, None, True, ones),
            lambda: e.step([StepItem(slot, [1], [0])], greedy(), None, True, ones[:, 1:]),
            lambda: e.step([StepItem(slot, [1], [0])], greedy(), None, True, np.ones((2, e.vocab), dtype=bool)),
            lambda: e.step([StepItem(slot, [1], [0])], greedy(), None, True, ones.astype(np.float32)),
            lambda: Engine.from_folder(model_folder("C"), head="int4"),
            lambda: Engine.from_folder(model_folder("C"), head="bfloat16")):
        with pytest.raises(InvalidArgError):
            call()
    assert e.sequence_length(slot) == 0 and tracked.sequence_length(other) == 0


# ---------------------------------------------------------------- the output matrix in four bits
def hidden_rows(name, toks):
    """The rows that meet the output matrix, 64-bit: the plain model with an identity in its place."""
    folder = model_folder(name)
    c, w = P.read_config(folder), dict(plain_weights(folder))
    head = w["lm_head.weight"] if not TINY[name]["tie_word_embeddings"] else w["model.embed_tokens.weight"]
    w["lm_head.weight"] = torch.eye(TINY[name]["hidden_size"], dtype=torch.float64)
    return P.forward_logits(dict(c, tie_word_embeddings=False), w, toks), head


@pytest.mark.parametrize("format", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["A", "B", "C"])
def test_logits_through_an_output_matrix_in_four_bits(name, dtype, format):
    """The engine's rows differ from the exact ones by their rounding, which now and then moves a value across the border between two codes, a step of at
    most a quarter of it where it is not small.  32-bit rows (2e-5) cross in one value in 10^4: 1e-2 of the result at most.  Bfloat16 rows (8e-3, as
    helpers.py measures them) cross in one in twenty, sqrt(1/20) / 4 = 6e-2 of the result, beside 8e-3 of their own: 8e-2."""
    from libllm_b200.engine import StepItem
    toks = tokens_for(name, 70, 13)
    rows, head = hidden_rows(name, toks)
    ref = Q.values(rows, format) @ Q.values(head, format).T
    bare = rows @ head.T
    e = engine(name, dtype, head=format)
    assert e.info()["head"] == format
    slot = e.open_sequence()
    got = [torch.from_numpy(e.step([StepItem(slot, toks[:60], list(range(60)))]).copy())]
    for t in toks[60:]:
        got.append(torch.from_numpy(e.step([StepItem(slot, [t], [0])]).copy()))
    got = torch.cat(got)
    assert rms_err(got, ref) < (1e-2 if dtype == "float32" else 8e-2)
    assert rms_err(got, ref) < rms_err(ref, bare), "nearer to the matrix in four bits than that is to the one it came from"


def test_the_whole_output_end_together():
    """Four-bit output matrix, penalties, bias and mask, drawn with temperature, in captured steps and in ones that are not: the same tokens."""
    from libllm_b200.engine import SamplingParams, StepItem
    rng = np.random.default_rng(6)
    s = SamplingParams(0.8, 20, 0.9, 1.2, 0.1, 0.1, {5: 1.0, 6: -1.0})
    masks = rng.random((9, 2, TINY["B"]["vocab_size"])) < 0.3
    uniforms = rng.random((9, 2))
    drawn = []
    for graphs in (True, False):
        e = engine("B", "bfloat16", head="nvfp4", track_history=True, use_graphs=graphs)
        slots = [e.open_sequence(), e.open_sequence()]
        tokens = [tokens_for("B", 9, 14), tokens_for("B", 21, 15)]
        mine = []
        for i in range(9):
            _, t = e.step([StepItem(q, t, [len(t) - 1]) for q, t in zip(slots, tokens)], s, uniforms[i], False, masks[i])
            assert all(masks[i, r, x] for r, x in enumerate(t))
            tokens = [[int(x)] for x in t]
            mine.append(tokens)
        drawn.append(mine)
        e.synchronize()
        e.cache_check()
    assert drawn[0] == drawn[1]


def test_the_command_line_takes_penalties_and_an_output_matrix_in_four_bits():
    """``bin/llm generate`` draws what Model.generate draws, and something else without penalties."""
    import os
    import subprocess
    from libllm_b200 import Model
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    folder, prompt = model_folder("C"), [5, 9, 2, 9]

    def by_command(*flags):
        out = subprocess.run([os.path.join(root, "bin", "llm"), "generate", "-m", folder, "--prompt-ids", ",".join(map(str, prompt)), "--max-new-tokens", "24",
                              "--temperature", "0", "--dtype", "float32", "--no-stop", "--max-tokens", "2048", *flags], capture_output=True, text=True, timeout=600)
        assert out.returncode == 0, out.stderr
        return [int(t) for t in out.stdout.strip().splitlines()[-1].split(",")]

    m = Model(folder, dtype="float32", max_tokens=2048, head="nvfp4", track_history=True)
    want = [m.generate([prompt], 24, temperature=0.0, stop_token_ids=[], **kw)[0]
            for kw in ({}, dict(repetition_penalty=1.5, presence_penalty=0.5, frequency_penalty=0.25))]
    assert want[0] != want[1]
    assert by_command("--head", "nvfp4") == want[0]
    assert by_command("--head", "nvfp4", "--repetition-penalty", "1.5", "--presence-penalty", "0.5", "--frequency-penalty", "0.25") == want[1]
    bad = subprocess.run([os.path.join(root, "bin", "llm"), "generate", "-m", folder, "--prompt-ids", "1,2", "--head", "fp4"], capture_output=True, text=True, timeout=600)
    assert bad.returncode != 0 and "fp4" in bad.stderr


def test_other_penalties_take_no_other_graphs():
    """Every step may bring penalties of its own: a captured step reads them from its descriptor."""
    e = engine(track_history=True, max_slots=4)
    seqs = [Sequence(e.open_sequence()) for _ in range(2)]
    drawn = run(e, seqs, [tokens_for("C", 12, 21), tokens_for("C", 5, 22)], greedy(repetition_penalty=1.3))
    before = e.info()["graphs_captured"]
    for i in range(10):
        s = greedy(repetition_penalty=1.0 + 0.05 * (i + 1), presence_penalty=0.01 * i, frequency_penalty=0.02 * (10 - i))
        drawn = run(e, seqs, [[t] for t in drawn], s)
    assert e.info()["graphs_captured"] - before == 2, "two graphs of the shape take turns, whatever the penalties"
    for s in (greedy(), greedy(presence_penalty=0.7), greedy(), greedy(repetition_penalty=0.8)):
        drawn = run(e, seqs, [[t] for t in drawn], s)
    assert e.info()["graphs_captured"] - before == 4, "two more of steps without penalties"


def test_operators_without_the_torch_binding(monkeypatch):
    """The same results by way of ctypes where the binding cannot be had."""
    from libllm_b200.csrc import ops
    from libllm_b200.errors import ExtensionError

    def fails():
        raise ExtensionError("no C++ compiler found")

    g = torch.Generator().manual_seed(30)
    x, w = (torch.randn(n, 300, generator=g).to(torch.bfloat16).cuda() for n in (5, 70))
    logits, history = torch.randn(3, 500, generator=g).cuda(), torch.randint(0, 500, (3, 40), generator=g).int().cuda()
    lengths = torch.tensor([40, 0, 17], dtype=torch.int32).cuda()

    def all_of_them():
        qx, qw = ops.fp4_quantize(x), ops.fp4_quantize(w)
        return [qx.codes, qx.row_scale, ops.fp4_dequantize(qw), ops.fp4_gemm(qx, qw), ops.fp4_gemm(qx, qw, out_dtype=torch.bfloat16),
                ops.adjust_logits(logits, history=history, lengths=lengths, repetition=1.5, presence=0.25)]

    want = all_of_them()
    monkeypatch.setattr(ops, "_quick", {})
    monkeypatch.setattr(ops, "_binding", [], raising=False)
    monkeypatch.setattr(ops.build, "load_binding", fails)
    assert all(torch.equal(a, b) for a, b in zip(want, all_of_them()))
    assert ops._binding == [None]


@pytest.mark.parametrize("graphs", [True, False])
def test_one_place_wanted_twice_in_a_step_of_single_tokens(graphs):
    """Two draws from the same logits, each with its own uniform number and mask, and the items behind keep theirs."""
    from libllm_b200.engine import SamplingParams, StepItem
    e = engine(use_graphs=graphs, track_history=True)
    V = e.vocab
    slots = [e.open_sequence() for _ in range(3)]
    for q in slots:
        e.step([StepItem(q, tokens_for("C", 4 + q, 31 + q), [])])
    items = [StepItem(slots[0], [5], [0, 0]), StepItem(slots[1], [6], [0]), StepItem(slots[2], [7], [0, 0, 0])]
    masks = np.zeros((6, V), dtype=bool)
    only = [3, V - 1, 40, 31, 32, 0]
    masks[np.arange(6), only] = True
    logits, drawn = e.step(items, greedy(repetition_penalty=1.2), None, True, masks)
    assert drawn.tolist() == only
    assert np.array_equal(logits[0], logits[1]) and np.array_equal(logits[3], logits[4]) and np.array_equal(logits[3], logits[5])
    assert not np.array_equal(logits[1], logits[2]) and not np.array_equal(logits[2], logits[3])
    # without sampling, and by uniform numbers
    plain = e.step([StepItem(slots[1], [9], [0, 0]), StepItem(slots[0], [8], [0])])
    assert np.array_equal(plain[0], plain[1]) and not np.array_equal(plain[1], plain[2])
    s = SamplingParams(1.0, 0, 1.0)
    u = [0.1, 0.9, 0.4]
    logits, drawn = e.step([StepItem(slots[1], [9], [0, 0]), StepItem(slots[0], [8], [0])], s, u)
    p = np.exp(logits.astype(np.float64) - logits.max(axis=1, keepdims=True))
    cdf = (p / p.sum(axis=1, keepdims=True)).cumsum(axis=1)
    for r, t in enumerate(drawn):
        low, high = (cdf[r, t - 1] if t else 0.0), cdf[r, t]
        assert low - 1e-5 <= u[r] <= high + 1e-5             # a draw's sums round by (V / 1024 + 50) 2^-24 = 3e-6 at most


@pytest.mark.parametrize("graphs", [True, False])
def test_a_token_fed_by_its_row_is_the_one_that_the_last_sampled_step_drew(graphs):
    """Whichever call ran that step, and also where not every item of it drew: the same logits, histories and draws as with the tokens' ids."""
    from libllm_b200.engine import StepItem
    s = greedy(repetition_penalty=1.4, presence_penalty=0.3, frequency_penalty=0.1)
    prompts = [tokens_for("C", n, 50 + n) for n in (9, 4, 6)]
    got = []
    for by_row in (False, True):
        e = engine(use_graphs=graphs, track_history=True)
        slots = [e.open_sequence() for _ in prompts]
        out = []

        def step(tokens, want, rows=None):
            items = [StepItem(q, t if rows is None or rows[i] is None or not by_row else [0], [len(t) - 1] if want[i] else [],
                              None if rows is None or not by_row else rows[i]) for i, (q, t) in enumerate(zip(slots, tokens))]
            logits, drawn = e.step(items, s)
            out.append((logits.copy(), drawn.tolist()))
            return [int(t) for t in drawn]

        d = step(prompts, [True, True, True])
        d = step([[t] for t in d], [True, True, True], [0, 1, 2])
        d2 = step([[t] for t in d], [False, True, True], [0, 1, 2])        # rows 0 and 1 are the second's and the third's now
        d3 = step([[7], [d2[0]], [d2[1]]], [True, False, True], [None, 0, 1])
        d4 = step([[d3[0]], [8, 9], [d3[1]]], [True, True, True], [0, None, 1])
        step([[t] for t in d4], [True, True, True], [0, 1, 2])
        got.append(out)
    for (la, da), (lb, db) in zip(*got):
        assert da == db and np.array_equal(la, lb)
