"""Rows with min-p in the sampler, on the host: which kernel takes which rows, and what goes up."""

import pytest
import torch

from somi_inference_b200.sampling import Sampler, SamplingParams
from tests import draw_plain
from tests.plain import sampler_plain
from tests.plain.host_ops import HostOps


class Ops(HostOps):
    """The plain kernels, and notes of their calls."""

    def __init__(self):
        super().__init__()
        self.sampled, self.drawn = [], []

    def uniform(self, seed, counter):
        return sampler_plain.uniform(seed, counter)

    def sample(self, logits, temperature, *rest):
        self.sampled.append(temperature.tolist())
        super().sample(logits, temperature, *rest)

    def draw_tokens(self, logits, uniform, temperature, top_k, top_p, min_p, out, prob=None, penalty=None, hist_off=None,
                    hist_tok=None):
        self.drawn.append(uniform.tolist())
        for r in range(logits.shape[0]):
            row = logits[r]
            if penalty is not None:
                row = draw_plain.penalised(row, float(penalty[r]), hist_tok[int(hist_off[r]):int(hist_off[r + 1])].long())
            tokens, p = draw_plain.draw(row, uniform[r].reshape(-1), float(temperature[r]), int(top_k[r]), float(top_p[r]), float(min_p[r]))
            out[r] = tokens.view(out[r].shape)
            if prob is not None:
                prob[r] = p.view(out[r].shape)


@pytest.fixture
def uploads(monkeypatch):
    """Every copy to a device, and whether it waits for the stream."""
    calls, inner, make = [], torch.Tensor.to, torch.tensor

    def to(self, *a, **k):
        if a and isinstance(a[0], (torch.device, str)) or "device" in k:
            calls.append(bool(k.get("non_blocking")))
        return inner(self, *a, **k)

    def tensor(*a, **k):
        if k.get("device") is not None:
            calls.append(False)
        return make(*a, **k)

    monkeypatch.setattr(torch.Tensor, "to", to)
    monkeypatch.setattr(torch, "tensor", tensor)
    return calls


def rows(n, seed=0):
    return torch.randn(n, 61, generator=torch.Generator().manual_seed(seed)) * 3


PLAIN = SamplingParams(temperature=0.9, top_k=20)
CUT = SamplingParams(temperature=0.9, min_p=0.05, top_p=0.9)
PENALISED = SamplingParams(temperature=1.1, min_p=0.02, repetition_penalty=1.5)
GREEDY = SamplingParams(temperature=0.0, min_p=0.5)


def test_rows_that_all_have_min_p_are_one_kernel_and_one_copy(uploads):
    ops = Ops()
    s = Sampler(ops, "cpu")
    s.sample(rows(3), [CUT] * 3, [4, 0, 2 ** 32 + 1], [5, 2 ** 64 + 6, 7])
    assert ops.sampled == [] and uploads == [True]
    want = [sampler_plain.uniform(5, 4), sampler_plain.uniform(6, 0), sampler_plain.uniform(7, 1)]
    assert ops.drawn == [want] and s.h2d_bytes_last >= 4 * 5 * 3


@pytest.mark.parametrize("params", [[PLAIN, CUT, PENALISED, GREEDY, PLAIN], [CUT, GREEDY], [PENALISED, PLAIN, PLAIN], [PENALISED]])
def test_mixed_rows_draw_as_they_do_alone_and_nothing_waits(uploads, params):
    ops = Ops()
    s = Sampler(ops, "cpu")
    n = len(params)
    x, counters, seeds = rows(n, n), list(range(n)), [100 + 3 * i for i in range(n)]
    histories = [[i, 5, i, 30 + i] for i in range(n)]
    together = s.sample(x, params, counters, seeds, histories)
    assert uploads == [True]
    cut = [i for i, p in enumerate(params) if p.min_p and p.temperature]
    # the usual kernel spends nothing on rows that it does not decide
    assert [[t > 0 for t in c] for c in ops.sampled] == ([[i not in cut and params[i].temperature > 0 for i in range(n)]] if len(cut) < n else [])
    for i, p in enumerate(params):
        assert s.sample(x[i:i + 1], [p], counters[i:i + 1], seeds[i:i + 1], histories[i:i + 1]).tolist() == [int(together[i])]
    for i in cut:
        p, row = params[i], x[i]
        if p.repetition_penalty != 1.0:
            row = draw_plain.penalised(row, p.repetition_penalty, sorted(set(histories[i])))
        u = torch.tensor([sampler_plain.uniform(seeds[i], counters[i])])
        want, _ = draw_plain.draw(row, u, *(float(torch.tensor(v)) if v != p.top_k else v for v in (p.temperature, p.top_k, p.top_p, p.min_p)))
        assert int(together[i]) == int(want[0])


def test_draws_from_given_numbers_are_one_copy(uploads):
    s = Sampler(Ops(), "cpu")
    u = torch.rand(2, 4, generator=torch.Generator().manual_seed(1))
    tokens, prob = s.draw(rows(2), [CUT, PLAIN], u)
    assert uploads == [True] and tokens.shape == prob.shape == (2, 4) and (prob > 0).all()
    assert s.draw(rows(2), [CUT, PLAIN], u, probabilities=False)[1] is None
