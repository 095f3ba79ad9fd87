"""What `CudaOps.draw_tokens` refuses before it launches anything, without a GPU."""

import ctypes

import pytest
import torch

from somi_inference_b200.ops import KernelError, cuda


class OnDevice(torch.Tensor):
    """A CPU tensor that the host side takes for one of device 0's."""
    is_cuda = True

    def get_device(self):
        return 0


@pytest.fixture
def ops(monkeypatch):
    table = cuda.CudaOps.__new__(cuda.CudaOps)
    table.launches, table._device_index, table.calls = 0, 0, []
    table._draw = lambda *a: table.calls.append(a) or 0
    table._stream = lambda: ctypes.c_void_p(0)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    return table


def arguments(**changed):
    rows, V = 3, 100
    a = dict(logits=torch.zeros(rows, V), uniform=torch.zeros(rows, 2), temperature=torch.ones(rows),
             top_k=torch.zeros(rows, dtype=torch.int32), top_p=torch.ones(rows), min_p=torch.zeros(rows),
             out=torch.zeros(rows, 2, dtype=torch.int32))
    a.update(changed)
    return {n: t.as_subclass(OnDevice) if isinstance(t, torch.Tensor) else t for n, t in a.items()}


HISTORY = dict(penalty=torch.ones(3), hist_off=torch.zeros(4, dtype=torch.int32), hist_tok=torch.zeros(1, dtype=torch.int32))


def test_consistent_calls_launch(ops):
    ops.draw_tokens(**arguments())
    ops.draw_tokens(**arguments(uniform=torch.zeros(3), out=torch.zeros(3, dtype=torch.int32), prob=torch.zeros(3)))
    ops.draw_tokens(**arguments(logits=torch.zeros(3, 200)[:, :100], **HISTORY))
    ops.draw_tokens(**arguments(logits=torch.zeros(3, 100).bfloat16()))
    assert [c[1:7:1][:4] for c in ops.calls] == [(0, 100, 3, 100), (0, 100, 3, 100), (0, 200, 3, 100), (1, 100, 3, 100)]
    assert [c[6] for c in ops.calls] == [2, 1, 2, 2] and ops.launches == 4
    assert [c[11] is None for c in ops.calls] == [True, True, False, True]
    assert [c[15] is None for c in ops.calls] == [True, False, True, True]


@pytest.mark.parametrize("changed", [
    dict(logits=torch.zeros(100)),
    dict(logits=torch.zeros(100, 3).t()),
    dict(logits=torch.zeros(3, 100).half()),
    dict(uniform=torch.zeros(2, 2)),
    dict(uniform=torch.zeros(3, 2, 1), out=torch.zeros(3, 2, 1, dtype=torch.int32)),
    dict(uniform=torch.zeros(3, 4)[:, ::2]),
    dict(uniform=torch.zeros(3, 2, dtype=torch.float64)),
    dict(out=torch.zeros(3, 2)),
    dict(out=torch.zeros(3, 1, dtype=torch.int32)),
    dict(prob=torch.zeros(3)),
    dict(prob=torch.zeros(3, 2, dtype=torch.int32)),
    dict(temperature=torch.ones(2)),
    dict(top_k=torch.zeros(3)),
    dict(top_k=torch.zeros(3, dtype=torch.int64)),
    dict(top_p=torch.ones(3, dtype=torch.float64)),
    dict(min_p=torch.ones(6)[::2]),
    dict(penalty=torch.ones(3)),
    dict(HISTORY, hist_off=torch.zeros(3, dtype=torch.int32)),
    dict(HISTORY, hist_tok=torch.zeros(1, dtype=torch.int64)),
    dict(HISTORY, logits=torch.zeros(3, 100).bfloat16()),
])
def test_refusals(ops, changed):
    with pytest.raises((KernelError, TypeError)):
        ops.draw_tokens(**arguments(**changed))
    assert not ops.calls and ops.launches == 0


@pytest.mark.parametrize("dtype,most", [(torch.float32, 786432), (torch.bfloat16, 2 ** 20 - 1)])
def test_a_vocabulary_that_is_too_large_is_named(ops, dtype, most):
    one = {n: torch.ones(1) for n in ("uniform", "temperature", "top_p", "min_p")}
    one.update(top_k=torch.zeros(1, dtype=torch.int32), out=torch.zeros(1, dtype=torch.int32))
    ops.draw_tokens(**arguments(logits=torch.zeros(1, most, dtype=dtype), **one))
    assert len(ops.calls) == 1
    with pytest.raises(KernelError, match=str(most)):
        ops.draw_tokens(**arguments(logits=torch.zeros(1, most + 1, dtype=dtype), **one))
    assert len(ops.calls) == 1


def test_a_request_with_min_p_and_too_large_a_vocabulary_is_refused_before_it_runs():
    from types import SimpleNamespace
    from somi_inference_b200 import LLM, SamplingParams
    llm = LLM.__new__(LLM)
    llm._next_request_id = 0
    for size, refused in ((786432, False), (786433, True)):
        llm.engine = SimpleNamespace(ops=SimpleNamespace(DRAW_MAX_VOCABULARY=cuda.CudaOps.DRAW_MAX_VOCABULARY),
                                     spec=SimpleNamespace(vocab_size=size))
        for sp in (SamplingParams(), SamplingParams(min_p=0.5, temperature=0.0)):
            assert llm.make_request([1], max_new_tokens=1, sampling_params=sp).sampling_params is sp
        if refused:
            with pytest.raises(ValueError, match="786432"):
                llm.make_request([1], max_new_tokens=1, sampling_params=SamplingParams(min_p=0.5))
        else:
            llm.make_request([1], max_new_tokens=1, sampling_params=SamplingParams(min_p=0.5))


def test_a_tensor_of_the_host_or_another_device_is_refused(ops):
    a = arguments()
    a["top_p"] = torch.ones(3)
    with pytest.raises(KernelError):
        ops.draw_tokens(**a)
    ops._device_index = 1
    with pytest.raises(KernelError, match="device"):
        ops.draw_tokens(**arguments())
    assert not ops.calls


def test_what_the_launcher_refuses_is_an_error(ops):
    ops._draw = lambda *a: cuda.ERR_UNSUPPORTED
    with pytest.raises(KernelError, match="not supported"):
        ops.draw_tokens(**arguments())


@pytest.mark.parametrize("value", [-0.1, 1.5, float("nan")])
def test_min_p_has_a_range(value):
    from somi_inference_b200 import SamplingParams
    with pytest.raises(ValueError):
        SamplingParams(min_p=value)


def test_the_command_takes_min_p():
    from somi_inference_b200.entrypoints.generate import parse_args
    assert parse_args(["--model-name", "m", "--prompt", "p", "--min-p", "0.2"]).min_p == 0.2
