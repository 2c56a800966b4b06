"""The output end of a decoding step as measurable cases: rows are brought into four bits, multiplied by a matrix that is held in
four bits, and the logits that come out are changed by what a request asks for before a token is drawn.

A case's ``op`` says which operator one pass runs:

* ``quantise``: rows into microscaled four-bit floating point (a value is one of +-{0, .5, 1, 1.5, 2, 3, 4, 6} times its block's scale
  times its row's), and the values that they then stand for;
* ``product``: rows of activations, brought into four bits within the call, times a matrix that was brought into four bits once;
* ``adjust``: penalties for what a sequence has said, a bias per token, a mask of allowed tokens, applied to rows of logits.

Formats: ``nvfp4`` has blocks of 16 along a row, scales of 8 bits (e4m3) and a power of two per row; ``mxfp4`` has blocks of 32 and
powers of two as scales.  Sizes are the benchmark's (hidden 2,048, 8,192 features, 128,256 tokens) or generic."""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

BLOCK = dict(nvfp4=16, mxfp4=32)
TYPES = dict(f32=torch.float32, bf16=torch.bfloat16)
MOST_VALUES = 128256 * 2048            # of one matrix: the listed output matrix
MOST_PRODUCTS = 8192 ** 3
MOST_LOGITS = 64 * 128256


def listed():
    return [
        # hidden rows of a step of eight requests, on their way to the output matrix
        dict(name="quantise 8x2048", op="quantise", rows=8, cols=2048, format="nvfp4", x="bf16", values="bf16", strided=False),
        # 32-bit rows of an odd width, cut out of wider ones
        dict(name="quantise 333x1111", op="quantise", rows=333, cols=1111, format="mxfp4", x="f32", values="f32", strided=True),
        # a prompt step's activations of 8,192 features
        dict(name="quantise 4096x8192", op="quantise", rows=4096, cols=8192, format="mxfp4", x="bf16", values="bf16", strided=False),
        # an output matrix of 128,256 tokens when it is loaded
        dict(name="quantise 128256x2048", op="quantise", rows=128256, cols=2048, format="nvfp4", x="bf16", values="bf16", strided=False),
        # a projection of one request's token
        dict(name="product 1x2048x2048", op="product", tokens=1, rows=2048, cols=2048, format="nvfp4", out="bf16"),
        # logits of a step of eight requests
        dict(name="product 8x128256x2048", op="product", tokens=8, rows=128256, cols=2048, format="nvfp4", out="f32"),
        # nothing a multiple of anything: a short prompt, a vocabulary that was never padded
        dict(name="product 37x1999x1500", op="product", tokens=37, rows=1999, cols=1500, format="mxfp4", out="bf16"),
        # a prompt of 2,048 tokens through a stacked gate and up matrix
        dict(name="product 2048x16384x2048", op="product", tokens=2048, rows=16384, cols=2048, format="nvfp4", out="bf16"),
        # a large prompt step through a wide square matrix
        dict(name="product 8192x8192x8192", op="product", tokens=8192, rows=8192, cols=8192, format="mxfp4", out="bf16"),
        # one request, a short conversation so far, penalties alone
        dict(name="adjust 1x128256", op="adjust", rows=1, vocab=128256, longest=512, penalties=True, bias="none", masked=False, strided=False),
        # seven requests with long histories over an odd vocabulary, rows cut out of wider ones
        dict(name="adjust 7x50257", op="adjust", rows=7, vocab=50257, longest=20000, penalties=True, bias="rows", masked=False, strided=True),
        # a full batch that uses everything: penalties, one bias for all, a grammar's mask per row
        dict(name="adjust 64x128256", op="adjust", rows=64, vocab=128256, longest=4096, penalties=True, bias="one", masked=True, strided=False),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over the logarithm; half of them pulled to a round one."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if n >= 64 and rng.random() < 0.5:
        n = n // 32 * 32
    return max(low, min(high, n))


def draw(rng):
    op = rng.choice(["quantise", "quantise", "product", "product", "adjust"])
    format = rng.choice(["nvfp4", "mxfp4"])
    if op == "quantise":
        cols = _spread(rng, 1, 16384)
        return dict(op=op, rows=_spread(rng, 1, min(131072, MOST_VALUES // cols)), cols=cols, format=format, x=rng.choice(["bf16", "bf16", "f32"]),
                    values=rng.choice(["bf16", "f32"]) if cols <= 4096 else "bf16", strided=rng.random() < 0.3)
    if op == "product":
        cols = _spread(rng, 16, 16384)
        tokens = _spread(rng, 1, 8192)
        return dict(op=op, tokens=tokens, rows=_spread(rng, 1, min(131072, MOST_VALUES // cols, MOST_PRODUCTS // (cols * tokens))), cols=cols,
                    format=format, out=rng.choice(["bf16", "f32"]))
    vocab = _spread(rng, 100, 160000)
    return dict(op=op, rows=_spread(rng, 1, max(1, min(256, MOST_LOGITS // vocab))), vocab=vocab, longest=_spread(rng, 1, 32768),
                penalties=rng.random() < 0.8, bias=rng.choice(["none", "one", "rows"]), masked=rng.random() < 0.6, strided=rng.random() < 0.3)


# ---------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 2 + 1)


def _activations(rows, cols, type, strided, gen):
    """Rows as a norm leaves them: bell-shaped, a few channels much larger than the rest, some rows small, a row of zeros among many."""
    wide = cols + 24 if strided else cols
    x = torch.randn(rows, wide, device="cuda", generator=gen)
    x *= torch.where(torch.rand(wide, device="cuda", generator=gen) < 0.01, 20.0, 1.0)
    x *= torch.exp2(torch.randint(-6, 3, (rows, 1), device="cuda", generator=gen).float())
    if rows > 100:
        x[rows // 2] = 0
    return x.to(TYPES[type])[:, :cols]


def _matrix(rows, cols, gen):
    return (torch.randn(rows, cols, device="cuda", generator=gen) * 0.02).to(torch.bfloat16)


def _histories(case, gen):
    """Token ids that repeat as words do (small ids much more often); the first half of each sequence is its prompt, stored as ~id."""
    rows, vocab, longest = case["rows"], case["vocab"], case["longest"]
    places = rows + 3                                               # more places than rows: sequences come and go
    ids = (vocab * torch.rand(places, longest, device="cuda", generator=gen) ** 4).int().clamp_(max=vocab - 1)
    slots = torch.randperm(places, device="cuda", generator=gen)[:rows].int()
    lengths = torch.randint(0, longest + 1, (rows,), device="cuda", generator=gen).int()
    lengths[rows // 2] = longest
    prompt = torch.zeros(places, dtype=torch.int32, device="cuda")
    prompt[slots.long()] = lengths // 2
    at = torch.arange(longest, device="cuda")
    return torch.where(at < prompt[:, None], ~ids, ids), slots, lengths


def prepare(case, seed):
    gen = _generator(seed)
    state = dict(case=case)
    if case["op"] == "quantise":
        state["x"] = _activations(case["rows"], case["cols"], case["x"], case["strided"], gen)
    elif case["op"] == "product":
        state["x"] = _activations(case["tokens"], case["cols"], "bf16", False, gen)
        w = _matrix(case["rows"], case["cols"], gen)
        if own:                                                     # a matrix is brought into four bits once, when it is loaded
            from libllm_b200.csrc import ops
            state["w"] = ops.fp4_quantize(w, case["format"])
        else:
            state["w"] = _four_bits(w, case["format"])
    else:
        rows, vocab = case["rows"], case["vocab"]
        wide = (vocab + 67) // 4 * 4 if case["strided"] else vocab
        state["logits"] = (3 * torch.randn(rows, wide, device="cuda", generator=gen))[:, :vocab]
        if case["penalties"]:
            state["history"], state["slots"], state["lengths"] = _histories(case, gen)
            state["repetition"] = 1 + 0.5 * torch.rand(rows, device="cuda", generator=gen)
            state["presence"] = torch.rand(rows, device="cuda", generator=gen)
            state["frequency"] = 0.2 * torch.rand(rows, device="cuda", generator=gen)
        if case["bias"] != "none":
            shape = (vocab,) if case["bias"] == "one" else (rows, vocab)
            some = torch.rand(shape, device="cuda", generator=gen) < 0.01
            state["bias"] = torch.where(some, 10 * torch.randn(shape, device="cuda", generator=gen), 0.0)
        if case["masked"]:
            words = (vocab + 31) // 32
            state["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (rows, words), device="cuda", generator=gen, dtype=torch.int64).int()
    return state


# ---------------------------------------------------------------- plain forms
def _two_to(exponent):
    """Powers of two, exact (exp2 and pow are off by a last bit here and there)."""
    return ((exponent.long() + 1023) << 52).view(torch.float64).float()


def _four_bits(x, format):
    """(codes [rows, blocks, block] as the eight magnitudes' numbers with a sign, scales [rows, blocks] and row scales [rows, 1] in 32 bits)."""
    rows, cols = x.shape
    block = BLOCK[format]
    x = torch.nn.functional.pad(x.float(), (0, -cols % block)).view(rows, -1, block)
    top = x.abs().amax(2)
    if format == "nvfp4":
        # The row's power of two puts its largest block's scale between 170 and 342, below e4m3's 448; no block that holds anything has a
        # scale below e4m3's smallest.
        exponent = torch.frexp(top.amax(1, keepdim=True)).exponent - 11
        row = torch.where(top.amax(1, keepdim=True) > 0, _two_to(exponent.clamp(min=-126)), 1.0)
        scale = (top / row / 6).to(torch.float8_e4m3fn).float()
        scale = torch.where(top > 0, scale.clamp(min=2.0 ** -9), 0.0)
        y = (x / row[:, :, None]).abs()
    else:
        # The block's power of two puts its largest value between 4 and 8; what lies above 6 becomes 6.
        row = torch.ones_like(top[:, :1])
        exponent = torch.where(top > 0, torch.frexp(top).exponent - 3, -127).clamp(min=-127)
        scale = _two_to(exponent)
        y = x.abs()
    s = scale[:, :, None]
    # halfway cases go to the even one of the two codes; a border times a scale is exact in 32 bits
    code = ((y > 0.25 * s).byte() + (y >= 0.75 * s).byte() + (y > 1.25 * s).byte() + (y >= 1.75 * s).byte() + (y > 2.5 * s).byte()
            + (y >= 3.5 * s).byte() + (y > 5 * s).byte())
    code = torch.where(s > 0, code, 0)
    return dict(codes=torch.where(x < 0, code + 8, code).byte(), scales=scale, row=row, cols=cols)


def _values(q):
    """What the codes stand for, 32-bit."""
    kinds = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, 0, -.5, -1, -1.5, -2, -3, -4, -6], device="cuda")
    rows = q["codes"].shape[0]
    return (kinds[q["codes"].int()] * q["scales"][:, :, None] * q["row"][:, :, None]).view(rows, -1)[:, :q["cols"]]


def _plain_quantise(state):
    return _values(_four_bits(state["x"], state["case"]["format"])).to(TYPES[state["case"]["values"]])


def _plain_product(state):
    x = _values(_four_bits(state["x"], state["case"]["format"]))
    return (x @ _values(state["w"]).T).to(TYPES[state["case"]["out"]])


def _plain_adjust(state):
    x = state["logits"]
    rows, vocab = x.shape
    if "history" in state:
        held = state["history"][state["slots"].long()]
        there = torch.arange(held.shape[1], device="cuda") < state["lengths"][:, None]
        ids = torch.where(held < 0, ~held, held).long()
        zeros = torch.zeros(rows, vocab, device="cuda")
        seen = zeros.scatter_add(1, ids, there.float()) > 0
        said = zeros.scatter_add(1, ids, (there & (held >= 0)).float())
        repetition = state["repetition"][:, None]
        x = torch.where(seen, torch.where(x > 0, x / repetition, x * repetition), x)
        x = torch.where(said > 0, x - (state["frequency"][:, None] * said + state["presence"][:, None]), x)
    if "bias" in state:
        x = x + state["bias"]
    if "allowed" in state:
        at = torch.arange(vocab, device="cuda")
        x = torch.where((state["allowed"][:, at >> 5] >> (at & 31)) & 1 == 1, x, -math.inf)
    return x


# ---------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if own:
        from libllm_b200.csrc import ops
        if case["op"] == "quantise":
            return ops.fp4_dequantize(ops.fp4_quantize(state["x"], case["format"]), TYPES[case["values"]])
        if case["op"] == "product":
            return ops.fp4_gemm(ops.fp4_quantize(state["x"], case["format"]), state["w"], out_dtype=TYPES[case["out"]])
        return ops.adjust_logits(state["logits"], history=state.get("history"), slots=state.get("slots"), lengths=state.get("lengths"),
                                 repetition=state.get("repetition", 1.0), presence=state.get("presence", 0.0),
                                 frequency=state.get("frequency", 0.0), bias=state.get("bias"), allowed=state.get("allowed"))
    if case["op"] == "quantise":
        return _plain_quantise(state)
    if case["op"] == "product":
        return _plain_product(state)
    return _plain_adjust(state)


def work(case):
    size = dict(f32=4, bf16=2)
    if case["op"] == "quantise":
        n = case["rows"] * case["cols"]
        return dict(bytes=n * (size[case["x"]] + size[case["values"]]), flops=4 * n)
    if case["op"] == "product":
        tokens, rows, cols, block = case["tokens"], case["rows"], case["cols"], BLOCK[case["format"]]
        held = rows * cols // 2 + rows * -(-cols // block) + 4 * rows
        return dict(bytes=held + 2 * tokens * cols + tokens * rows * size[case["out"]], flops=2 * tokens * rows * cols)
    rows, vocab = case["rows"], case["vocab"]
    bias = dict(none=0, one=vocab, rows=rows * vocab)[case["bias"]]
    history = rows * case["longest"] // 2 if case["penalties"] else 0           # lengths are even over 0 .. longest
    mask = rows * (vocab + 31) // 32 if case["masked"] else 0
    return dict(bytes=4 * (2 * rows * vocab + bias + history + mask), flops=3 * rows * vocab)


# ---------------------------------------------------------------- the definition in 64 bits
def _power_below(v, of_zero):
    """The largest power of two that is not above v > 0 (its fraction's bits cleared); `of_zero` for 0."""
    return torch.where(v > 0, (v.view(torch.int64) >> 52 << 52).view(torch.float64), of_zero)


def _exact_values(x, format):
    """What a row's values become: the nearest of what its block's scale can reach, halves to even."""
    rows, cols = x.shape
    block = BLOCK[format]
    full = -(-cols // block) * block
    v = torch.zeros(rows, full, dtype=torch.float64, device="cuda")
    v[:, :cols] = x.double()
    v = v.reshape(rows, full // block, block)
    largest = v.abs().max(dim=2, keepdim=True).values
    if format == "nvfp4":
        of_row = largest.max(dim=1, keepdim=True).values
        row = torch.clamp(_power_below(of_row, 1024.0) / 1024, min=2.0 ** -126)
        wanted = largest / (6 * row)
        step = torch.clamp(_power_below(wanted, 0.0), min=2.0 ** -6) / 8                            # e4m3: three bits behind the first, to 2^-9
        unit = torch.where(largest > 0, torch.clamp(torch.round(wanted / step) * step, min=2.0 ** -9), 1.0) * row
    else:
        unit = torch.clamp(_power_below(largest, 0.0) / 4, min=2.0 ** -127)
    a = v.abs() / unit
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).double()
    near = torch.clamp(torch.round(a / step) * step, max=6.0)
    return (torch.sign(v) * near * unit).reshape(rows, full)[:, :cols]


def exact(case, seed):
    gen = _generator(seed)
    if case["op"] == "quantise":
        return _exact_values(_activations(case["rows"], case["cols"], case["x"], case["strided"], gen), case["format"])
    if case["op"] == "product":
        x = _activations(case["tokens"], case["cols"], "bf16", False, gen)
        w = _matrix(case["rows"], case["cols"], gen)
        return _exact_values(x, case["format"]) @ _exact_values(w, case["format"]).T
    state = {k: v.cpu().numpy() if isinstance(v, torch.Tensor) else v for k, v in prepare(case, seed).items()}
    rows, vocab = case["rows"], case["vocab"]
    out = state["logits"].astype(np.float64)
    for r in range(rows):
        if case["penalties"]:
            ids = state["history"][state["slots"][r], :state["lengths"][r]]
            drawn = np.bincount(ids[ids >= 0], minlength=vocab)
            seen = np.bincount(np.where(ids < 0, -1 - ids, ids), minlength=vocab) > 0
            by = np.float64(state["repetition"][r])
            out[r, seen] = np.where(out[r, seen] > 0, out[r, seen] / by, out[r, seen] * by)
            out[r] -= np.float64(state["frequency"][r]) * drawn + np.float64(state["presence"][r]) * (drawn > 0)
        if case["bias"] != "none":
            out[r] += (state["bias"] if case["bias"] == "one" else state["bias"][r]).astype(np.float64)
        if case["masked"]:
            bits = np.unpackbits(state["allowed"][r].astype("<i4").view(np.uint8), bitorder="little")[:vocab]
            out[r, bits == 0] = -np.inf
    return torch.from_numpy(out)
