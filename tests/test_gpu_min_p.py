"""Rows with min-p do not make the host wait for the step in front of them."""

import pytest
import torch

from somi_inference_b200.sampling import Sampler, SamplingParams

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("which", ["some", "all"])
def test_sampling_returns_while_the_stream_is_busy(which):
    from somi_inference_b200.ops import cuda_ops
    s = Sampler(cuda_ops(), "cuda")
    g = torch.Generator().manual_seed(3)
    logits = (torch.randn(6, 32003, generator=g) * 3).cuda()
    cut, plain = SamplingParams(temperature=0.8, min_p=0.02), SamplingParams(temperature=0.8)
    params = [cut, plain, cut, SamplingParams(temperature=0.0), cut, plain] if which == "some" else [cut] * 6
    counters, seeds = list(range(6)), [11 * i for i in range(6)]
    want = s.sample(logits, params, counters, seeds).tolist()
    assert [s.sample(logits[i:i + 1], params[i:i + 1], counters[i:i + 1], seeds[i:i + 1]).item() for i in range(6)] == want
    a = torch.randn(8192, 8192, device="cuda", dtype=torch.bfloat16)
    b = torch.empty_like(a)
    torch.mm(a, a, out=b)
    torch.cuda.synchronize()
    for _ in range(100):                     # about 70 ms in front of the rows; the call takes well below one
        torch.mm(a, a, out=b)
    in_front = torch.cuda.Event()
    in_front.record()
    got = s.sample(logits, params, counters, seeds)
    waited = in_front.query()
    assert got.tolist() == want
    assert not waited
