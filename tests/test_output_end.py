"""What the operators of a step's output end refuse, told before anything is launched: on the CPU, where nothing could be."""
import pytest
import torch

from libllm_b200.csrc import ops
from libllm_b200.errors import ExtensionError, InvalidArgError, UnsupportedError

I32 = torch.int32


def matrix(rows, cols, format="nvfp4"):
    return ops.Fp4Matrix(rows, cols, format, "cpu")


@pytest.mark.parametrize("call", [
    lambda: ops.Fp4Matrix(4, 0, "nvfp4", "cpu"),
    lambda: ops.Fp4Matrix(-1, 4, "nvfp4", "cpu"),
    lambda: ops.Fp4Matrix(4, 64, "fp4", "cpu"),
    lambda: ops.fp4_quantize(torch.zeros(4, 64), "e2m1"),
    lambda: ops.fp4_quantize(torch.zeros(64)),
    lambda: ops.fp4_quantize(torch.zeros(64, 4).T),
    lambda: ops.fp4_quantize(torch.zeros(4, 64), "nvfp4", out=matrix(4, 63)),
    lambda: ops.fp4_quantize(torch.zeros(4, 64), "nvfp4", out=matrix(4, 64, "mxfp4")),
    lambda: ops.fp4_dequantize(matrix(4, 64), out=torch.zeros(4, 63)),
    lambda: ops.fp4_dequantize(matrix(4, 64), out=torch.zeros(1, 64).expand(4, 64)),
    lambda: ops.fp4_gemm(matrix(4, 64), matrix(4, 65)),
    lambda: ops.fp4_gemm(matrix(4, 64), matrix(4, 64, "mxfp4")),
    lambda: ops.fp4_gemm(matrix(4, 64), matrix(5, 64), out=torch.zeros(5, 4)),
    lambda: ops.fp4_gemm(matrix(4, 64), matrix(5, 64), out=torch.zeros(5, 4).T),
    lambda: ops.fp4_gemm(matrix(4, 64), matrix(5, 64), out=torch.zeros(1, 5).expand(4, 5)),
])
def test_matrices_in_four_bits(call):
    with pytest.raises(InvalidArgError):
        call()


@pytest.mark.parametrize("call", [
    lambda: ops.fp4_quantize(torch.zeros(4, 64, dtype=torch.float16)),
    lambda: ops.fp4_dequantize(matrix(4, 64), torch.float64),
    lambda: ops.fp4_gemm(matrix(4, 64), matrix(5, 64), out_dtype=torch.float16),
    lambda: ops.adjust_logits(torch.zeros(1, 5).expand(70000, 5)),
])
def test_types_and_sizes_that_are_not_taken(call):
    with pytest.raises(UnsupportedError):
        call()


@pytest.mark.parametrize("call", [
    lambda: ops.fp4_quantize(torch.zeros(4, 64)),
    lambda: ops.fp4_dequantize(matrix(4, 64)),
    lambda: ops.fp4_gemm(matrix(4, 64), matrix(5, 64)),
    lambda: ops.adjust_logits(torch.zeros(4, 64)),
])
def test_there_is_no_way_to_run_without_a_device(call):
    with pytest.raises(ExtensionError):
        call()


B, V = 3, 100
HISTORY, LENGTHS = torch.zeros(5, 20, dtype=I32), torch.zeros(B, dtype=I32)


@pytest.mark.parametrize("kw", [
    dict(logits=torch.zeros(B, V, dtype=torch.bfloat16)),
    dict(logits=torch.zeros(V)),
    dict(logits=torch.zeros(V, B).T),
    dict(out=torch.zeros(B, V + 1)),
    dict(out=torch.zeros(B, V, dtype=torch.bfloat16)),
    dict(out=torch.zeros(1, V).expand(B, V)),
    dict(history=HISTORY),
    dict(history=HISTORY.long(), lengths=LENGTHS),
    dict(history=HISTORY[0], lengths=LENGTHS),
    dict(history=HISTORY.T, lengths=LENGTHS),
    dict(history=HISTORY[:2], lengths=LENGTHS),
    dict(history=HISTORY, lengths=LENGTHS[:2]),
    dict(history=HISTORY, lengths=LENGTHS.long()),
    dict(history=HISTORY, lengths=LENGTHS, slots=LENGTHS.long()),
    dict(history=HISTORY, lengths=LENGTHS, slots=LENGTHS[:1]),
    dict(repetition=0.0),
    dict(repetition=-1.0),
    dict(repetition=float("inf")),
    dict(presence=float("nan")),
    dict(frequency=torch.zeros(B + 1)),
    dict(frequency=torch.zeros(B, dtype=torch.float64)),
    dict(bias=torch.zeros(V + 1)),
    dict(bias=torch.zeros(1, V)),
    dict(bias=torch.zeros(V, dtype=torch.bfloat16)),
    dict(bias=torch.zeros(V, B).T),
    dict(allowed=torch.zeros(3, dtype=I32)),
    dict(allowed=torch.zeros(B, 5, dtype=I32)),
    dict(allowed=torch.zeros(B, V, dtype=torch.bool)),
    dict(allowed=torch.zeros(4, B, dtype=I32).T),
])
def test_logits_and_what_goes_with_them(kw):
    kw = dict(kw)
    logits = kw.pop("logits", torch.zeros(B, V))
    with pytest.raises(InvalidArgError):
        ops.adjust_logits(logits, **kw)


@pytest.mark.parametrize("kw", [dict(repetition=1e39), dict(repetition=1e-46), dict(repetition=10 ** 39), dict(presence=-1e39), dict(frequency=1e300)])
def test_penalties_that_32_bits_do_not_hold(kw):
    with pytest.raises(InvalidArgError):
        ops.adjust_logits(torch.zeros(B, V), **kw)


def changed(**kw):
    q = matrix(4, 64)
    for name, v in kw.items():
        setattr(q, name, v)
    return q


@pytest.mark.parametrize("kw", [dict(data=matrix(4, 64).data[:-1]), dict(data=torch.zeros(2 * matrix(4, 64).nbytes, dtype=torch.uint8)[::2]),
                                dict(data=torch.zeros(matrix(4, 64).nbytes, dtype=torch.int8)), dict(rows=400), dict(cols=6400), dict(cols=0)])
def test_matrices_whose_memory_is_not_theirs(kw):
    rows, cols = kw.get("rows", 4), kw.get("cols", 64)
    calls = [lambda q: ops.fp4_dequantize(q), lambda q: ops.fp4_dequantize(q, out=torch.zeros(rows, cols)),
             lambda q: ops.fp4_gemm(q, ops.Fp4Matrix(3, max(cols, 1), "nvfp4", "cpu")),
             lambda q: ops.fp4_gemm(q, ops.Fp4Matrix(3, max(cols, 1), "nvfp4", "cpu"), out=torch.zeros(rows, 3)),
             lambda q: ops.fp4_gemm(ops.Fp4Matrix(3, max(cols, 1), "nvfp4", "cpu"), q),
             lambda q: ops.fp4_quantize(torch.zeros(rows, max(cols, 1)), out=q)]
    for call in calls:
        with pytest.raises(InvalidArgError):
            call(changed(**kw))


@pytest.mark.parametrize("error", [ExtensionError("no C++ compiler found"), PermissionError("the folder cannot be written")])
def test_without_the_torch_binding_calls_go_the_longer_way(error, monkeypatch, capsys):
    """Told once, tried once, and answered with None, upon which every operator goes through its own checks to the kernel."""
    class OnGpu:
        is_cuda = True

    tried = []

    def fails():
        tried.append(1)
        raise error

    monkeypatch.setattr(ops, "_quick", {})
    monkeypatch.setattr(ops, "_binding", [], raising=False)
    monkeypatch.setattr(ops.build, "load_binding", fails)
    for family, name in (("fp4", "fp4_quantize"), ("fp4", "fp4_gemm"), ("logits", "adjust_logits"), ("fp4", "fp4_quantize")):
        assert ops._quick_call(family, name, OnGpu())(1, 2, 3) is None
        assert ops._quick[name](4) is None
    assert len(tried) == 1 and capsys.readouterr().err.count(str(error)) == 1


def test_token_ids_of_a_bias():
    import numpy as np
    from libllm_b200.engine import SamplingParams
    for bias in ({1: 2}, {"1": 2}, {1.0: 2}, {np.int64(1): 2}, [(1, 2)], ((np.float32(1), 2.0),)):
        assert SamplingParams(logit_bias=bias).logit_bias == ((1, 2.0),)
    assert SamplingParams(logit_bias=None).logit_bias == () == SamplingParams(logit_bias={}).logit_bias
    for bias in ({1.7: 2.0}, [(np.float32(0.5), 1.0)], {-0.5: 1.0}):
        with pytest.raises(InvalidArgError):
            SamplingParams(logit_bias=bias)
