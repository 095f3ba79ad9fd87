"""Draws from given random numbers (`CudaOps.draw_tokens`) against 64 bits, token for token.

A sum of n weights that are rounded to multiples of 2^-44 is off by at most n 2^-45 (largest weight: 1), so a
number within that of a border could fall on either side: at most 1e-8 of all numbers for the vocabularies here.
The numbers are fixed by their seeds and none of them does."""

import pytest
import torch

from tests import draw_plain

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from somi_inference_b200.ops import cuda_ops
    return cuda_ops()


def check(ops, logits, settings, u, history=None, penalty=None):
    """`settings`: (temperature, top_k, top_p, min_p) of every row; `u` [rows, draws]."""
    dev = logits if logits.is_cuda else logits.cuda()
    rows = len(settings)
    cols = [torch.tensor(c) for c in zip(*settings)]
    extra = {}
    if penalty is not None:
        off = torch.tensor([0] + [len(h) for h in history]).cumsum(0)
        extra = dict(penalty=torch.tensor(penalty).cuda(), hist_off=off.int().cuda(),
                     hist_tok=torch.tensor([t for h in history for t in h] or [0]).int().cuda())
    out = torch.full(u.shape, -5, dtype=torch.int32, device="cuda")
    prob = torch.full(u.shape, -5.0, device="cuda")
    ops.draw_tokens(dev, u.cuda(), cols[0].float().cuda(), cols[1].int().cuda(), cols[2].float().cuda(),
                    cols[3].float().cuda(), out, prob=prob, **extra)
    host = dev.cpu().float()
    for r in range(rows):
        row = host[r] if penalty is None or penalty[r] == 1.0 else draw_plain.penalised(host[r], penalty[r], history[r])
        T, k, p, m = (float(torch.tensor(v, dtype=torch.float32)) if i != 1 else v for i, v in enumerate(settings[r]))
        tokens, probs = draw_plain.draw(row, u[r].reshape(-1), T, k, p, m)
        assert out[r].reshape(-1).cpu().tolist() == tokens.tolist(), (r, settings[r])
        # a weight and the mass are each off by 2^-45 n, the quotient is rounded once to float32
        assert torch.allclose(prob[r].reshape(-1).cpu(), probs, rtol=2.0 ** -22, atol=0), (r, settings[r])
    return out


SETTINGS = [(1.0, -1, 1.0, 0.0), (0.7, 20, 0.8, 0.05), (0.0, -1, 1.0, 0.0), (1.3, -1, 0.95, 0.0), (0.8, 50, 1.0, 0.0),
            (1.0, -1, 1.0, 0.02), (1.0, 1, 1.0, 0.0), (2.0, 1000, 0.5, 0.0), (0.3, 0, 0.99, 0.5), (5.0, -1, 0.999, 0.001),
            (1.0, 10 ** 9, 1.0, 1.0), (1.0, 7, 0.0, 0.0)]


def rows_of(n, V, seed, dtype=torch.float32, spread=2.2):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, V, generator=g) * spread
    for r in range(n):
        x[r, torch.randint(0, V, (min(V, 30),), generator=g)] += 3 + 8 * torch.rand(min(V, 30), generator=g)
    return x.to(dtype), torch.rand(n, 9, generator=g)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [1, 2, 31, 33, 517, 4095, 4097, 32003, 151936])
def test_rows_with_settings_of_their_own(ops, V, dtype):
    x, u = rows_of(len(SETTINGS), V, V, dtype)
    check(ops, x, SETTINGS, u)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_flat_rows(ops, dtype):
    """Nearly equal weights: a cut that lies among thousands of tokens."""
    x, u = rows_of(len(SETTINGS), 50000, 5, dtype, spread=0.05)
    check(ops, (x - x.clamp(min=1.0) + 1.0).to(dtype), SETTINGS, u)
    x = torch.randn(len(SETTINGS), 20001, generator=torch.Generator().manual_seed(1)).to(dtype)
    check(ops, x, [(50.0, k, p, m) for _, k, p, m in SETTINGS], u)


def test_a_mass_cut_among_a_whole_vocabulary(ops):
    """top-p alone, its cut among tens of thousands of kept tokens; zeros, masked and NaN logits among them, several maxima."""
    g = torch.Generator().manual_seed(30)
    x = torch.randn(10, 60001, generator=g)
    x[1, ::3] = 0.0
    x[1, 1::3] = -0.0
    x[2, ::2] = float("nan")
    x[3, ::2] = -float("inf")
    x[4] = (x[4] * 4).round() / 4            # few different values
    x[5] *= 12                               # most of the mass in a few, the cut in what vanishes
    x[6, 100:110] = 9.0
    x[7] = x[7].abs() * -1e-3
    x[8] = torch.linspace(-40, 0, 60001)[torch.randperm(60001, generator=g)]
    u = torch.rand(10, 20, generator=g)
    for dtype in (torch.float32, torch.bfloat16):
        for p in (0.5, 0.95, 0.999999):
            check(ops, x.to(dtype), [(1.0, -1, p, 0.0), (0.9, -1, p, 0.0), (1.0, 0, p, 0.2), (1.0, 70000, p, 0.0), (1.0, -1, p, 1e-3)] * 2, u)
    ops.check_errors()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_equal_logits_are_kept_by_their_index(ops, dtype):
    """Few different values, so every cut lies among equal ones: 3 values, and all equal."""
    g = torch.Generator().manual_seed(2)
    x = torch.randint(0, 3, (len(SETTINGS), 9001), generator=g).to(dtype)
    u = torch.rand(len(SETTINGS), 40, generator=g)
    check(ops, x, SETTINGS, u)
    check(ops, torch.zeros_like(x), [(1.0, 4500, 1.0, 0.0), (1.0, -1, 0.5, 0.0), (1.0, 9000, 0.25, 0.0), (1.0, 1, 0.5, 1.0),
                                     (0.5, 100, 0.75, 0.5), (9.0, -1, 0.125, 0.0)] * 2, u)


def test_zeros_of_both_signs_are_equal(ops):
    x = torch.zeros(2, 100)
    x[:, ::2] = -0.0
    u = torch.rand(2, 30, generator=torch.Generator().manual_seed(0))
    check(ops, x, [(1.0, 10, 1.0, 0.0), (0.0, -1, 1.0, 0.0)], u)


@pytest.mark.parametrize("settings", [(1.0, -1, 1.0, 0.0), (0.7, 5, 0.9, 0.1), (1.0, -1, 0.9, 0.0), (0.0, 3, 0.5, 0.5)])
def test_masked_rows_infinities_and_nan(ops, settings):
    inf, nan, low = float("inf"), float("nan"), torch.finfo(torch.float32).min
    g = torch.Generator().manual_seed(3)
    x = torch.randn(9, 5003, generator=g)
    x[0, 1:] = -inf
    x[1, :-1] = -inf
    x[2] = -inf                              # nothing left
    x[3, ::2] = nan
    x[4] = nan
    x[5, [7, 900, 5002]] = inf
    x[6, :5000] = low                        # a mask by the type's lowest value
    x[7] = low
    x[8, 17] = 3.4e38
    u = torch.rand(9, 12, generator=g)
    check(ops, x, [settings] * 9, u)


def test_a_range_of_temperatures(ops):
    x, u = rows_of(8, 3001, 11)
    check(ops, x, [(T, -1, 0.9, 0.0) for T in (1e-38, 1e-6, 1e-3, 0.05, 30.0, 1e4, 1e30, float("inf"))], u)


def test_numbers_at_the_ends(ops):
    x, _ = rows_of(4, 2003, 12)
    u = torch.tensor([[0.0, 2.0 ** -24, 1 - 2.0 ** -24, 0.5, 2.0 ** -126]] * 4)
    check(ops, x, [(1.0, -1, 1.0, 0.0), (0.7, 20, 0.8, 0.05), (1.0, 1, 1.0, 0.0), (1.0, -1, 0.9, 0.0)], u)


def test_numbers_outside_their_range_draw_a_kept_token(ops):
    x, _ = rows_of(1, 2003, 13)
    u = torch.tensor([[-1.0, 1.0, 7.0, float("nan"), float("inf")]])
    out, one = torch.zeros(1, 5, dtype=torch.int32, device="cuda"), torch.ones(1, device="cuda")
    ops.draw_tokens(x.cuda(), u.cuda(), one, (5 * one).int(), one, 0 * one, out)
    top = torch.topk(x[0], 5).indices.sort().values
    assert out[0].tolist() == [int(top[0]), int(top[-1]), int(top[-1]), int(top[0]), int(top[-1])]


def test_rows_that_lie_apart_and_begin_anywhere(ops):
    g = torch.Generator().manual_seed(14)
    for dtype in (torch.float32, torch.bfloat16):
        store = torch.randn(5 * 9011 + 3, generator=g).to(dtype).cuda()
        for first in (0, 1, 3):
            x = store[first:first + 5 * 9011].view(5, 9011)[:, :8999]
            check(ops, x, [SETTINGS[i] for i in (0, 1, 3, 5, 7)], torch.rand(5, 3, generator=g))


def test_one_draw_a_row_as_a_vector_and_many_rows(ops):
    x, _ = rows_of(300, 1500, 15)
    g = torch.Generator().manual_seed(15)
    u = torch.rand(300, generator=g)
    check(ops, x, (SETTINGS * 25), u)


def test_a_large_vocabulary(ops):
    g = torch.Generator().manual_seed(16)
    x = torch.randn(2, 450007, generator=g) * 3
    check(ops, x, [(1.0, -1, 1.0, 0.0), (1.0, -1, 0.9, 0.01)], torch.rand(2, 6, generator=g))
    check(ops, x.bfloat16(), [(1.0, 40, 1.0, 0.0), (1.0, -1, 0.7, 0.0)], torch.rand(2, 6, generator=g))


def test_repetition_penalty(ops):
    g = torch.Generator().manual_seed(17)
    x, u = rows_of(4, 4801, 17)
    history = [torch.randperm(4801, generator=g)[:n].tolist() for n in (0, 1, 200, 4801)]
    check(ops, x, [(1.0, -1, 1.0, 0.0), (0.7, 20, 0.9, 0.0), (0.0, -1, 1.0, 0.0), (1.0, -1, 0.9, 0.1)], u, history, [1.3, 1.0, 2.0, 0.7])


def test_equal_rows_give_equal_tokens_whatever_the_batch(ops):
    x, u = rows_of(1, 151936, 18)
    dev = x.cuda()

    def draw(n):
        one = torch.ones(n, device="cuda")
        out = torch.empty(n, 9, dtype=torch.int32, device="cuda")
        ops.draw_tokens(dev.expand(n, -1), u.cuda().repeat(n, 1), one, (0 * one).int(), 0.95 * one, 0.01 * one, out)
        return out
    alone = draw(1)
    assert all((draw(n) == alone).all() for n in (2, 9, 70))


def test_a_captured_call_reads_new_numbers_and_settings(ops):
    x, u = rows_of(2, 5000, 19)
    hold = dict(x=x.cuda(), u=u.cuda(), t=torch.ones(2, device="cuda"), k=torch.zeros(2, dtype=torch.int32, device="cuda"),
                p=torch.ones(2, device="cuda"), m=torch.zeros(2, device="cuda"))
    out = torch.empty(2, 9, dtype=torch.int32, device="cuda")
    ops.draw_tokens(*hold.values(), out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.draw_tokens(*hold.values(), out)
    y, v = rows_of(2, 5000, 20)
    hold["x"].copy_(y), hold["u"].copy_(v), hold["k"].fill_(9), hold["p"].fill_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    for r in range(2):
        assert out[r].tolist() == draw_plain.draw(y[r], v[r], 1.0, 9, 0.5, 0.0)[0].tolist()


def test_no_rows_or_draws_is_no_launch(ops):
    before = ops.launches
    f, i = torch.empty(0, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda")
    ops.draw_tokens(torch.empty(0, 9, device="cuda"), f, f, i, f, f, i)
    one = torch.ones(1, device="cuda")
    ops.draw_tokens(torch.empty(1, 9, device="cuda"), f.view(1, 0), one, one.int(), one, one, i.view(1, 0))
    assert ops.launches == before


@pytest.mark.parametrize("rows", [1, 13, 260])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_flat_rows_of_any_number_with_many_draws(ops, rows, dtype):
    """top-p alone among nearly equal weights: numbers fall on every part of a row, however many CTAs share it."""
    g = torch.Generator().manual_seed(rows)
    x = (torch.randn(rows, 70001, generator=g) * 0.7).to(dtype)
    u = torch.rand(rows, 33, generator=g)
    u[:, 0], u[:, 1] = 0.0, 1.0 - 2.0 ** -24
    settings = [(0.9, -1, (0.9, 0.3, 0.99)[r % 3], 0.0) for r in range(rows)]
    if rows < 260:
        check(ops, x, settings, u)
        return
    some = [0, 1, 2, 77, 128, 259]
    args = [torch.tensor(c).cuda() for c in zip(*settings)]
    out, prob = torch.empty(u.shape, dtype=torch.int32, device="cuda"), torch.empty(u.shape, device="cuda")
    ops.draw_tokens(x.cuda(), u.cuda(), args[0].float(), args[1].int(), args[2].float(), args[3].float(), out, prob=prob)
    alone = check(ops, x[some], [settings[r] for r in some], u[some])
    assert torch.equal(out[some], alone)
    ops.check_errors()


def test_two_calls_at_once(ops):
    g = torch.Generator().manual_seed(3)
    calls = []
    for i, (rows, V) in enumerate(((4, 152064), (60, 32000))):
        n = len(SETTINGS)
        cols = [torch.tensor([SETTINGS[(r + i) % n][c] for r in range(rows)]).cuda() for c in range(4)]
        calls.append((torch.randn(rows, V, generator=g).mul(3).cuda(), torch.rand(rows, 3, generator=g).cuda(), cols[0].float(),
                      cols[1].int(), cols[2].float(), cols[3].float()))

    def run(c):
        out, prob = torch.empty(c[1].shape, dtype=torch.int32, device="cuda"), torch.empty(c[1].shape, device="cuda")
        ops.draw_tokens(*c, out, prob=prob)
        return out, prob

    alone = [run(c) for c in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    got = []
    for _ in range(6):
        for c, s in zip(calls, streams):
            with torch.cuda.stream(s):
                got.append(run(c))
    torch.cuda.synchronize()
    for i, (out, prob) in enumerate(got):
        assert torch.equal(out, alone[i % 2][0]) and torch.equal(prob, alone[i % 2][1])
    ops.check_errors()


def test_counted_values_of_16_bits(ops):
    """Rows long enough for a CTA to count values, and what it does not count: NaN, zeros, values next to zero and far from it."""
    g = torch.Generator().manual_seed(40)
    V = 152064
    x = torch.randn(17, V, generator=g)
    x[1, ::2] = float("nan")
    x[2, ::3], x[2, 1::3] = 0.0, -0.0
    x[3] *= 2.0 ** -9                        # most of them below the least value that is counted
    x[4] *= 150                              # some above the largest
    x[5, ::2] = -float("inf")
    x[6] = (x[6] * 2).round() / 2            # few values, thousands of tokens each
    x[7] = 1.0
    x[8] = -300.0 + x[8]
    x[9, 100:200] = float("inf")
    x[10] = 2.0 ** -8 * (1 - 2 * torch.randint(0, 2, (V,), generator=g)) * (1 + torch.randint(0, 2, (V,), generator=g) / 128)
    x[11] = 256.0 - x[11].abs()
    x[12] = -x[12].abs()
    x[13] *= 5
    x = x.bfloat16()
    u = torch.rand(17, 12, generator=g)
    for p in (0.3, 0.97):
        check(ops, x, [((1.0, 0.6, 3.0)[r % 3], -1, p, 0.0 if r % 5 else 1e-4) for r in range(17)], u)
    ops.check_errors()


@pytest.mark.parametrize("dtype,code", [(torch.float32, 0), (torch.bfloat16, 1)])
def test_the_largest_vocabulary(ops, dtype, code):
    from somi_inference_b200.ops import KernelError
    V = ops.lib.somi_draw_max_vocabulary(code)
    assert V == ops.DRAW_MAX_VOCABULARY[dtype]
    g = torch.Generator().manual_seed(50)
    x = (torch.randn(4, V, generator=g) * 3).to(dtype)
    x[2:] = (x[2:].float() * 0.2).to(dtype)
    u = torch.rand(4, 5, generator=g)
    u[:, 0], u[:, 1] = 0.0, 1.0 - 2.0 ** -24
    check(ops, x, [(1.0, -1, 1.0, 0.0), (0.8, 40, 0.9, 0.05), (1.0, -1, 0.9, 0.0), (1.0, -1, 1.0, 0.01)], u)
    one = torch.ones(1, device="cuda")
    out = torch.full((1,), -5, dtype=torch.int32, device="cuda")
    with pytest.raises(KernelError, match="vocabular"):
        ops.draw_tokens(torch.zeros(1, V + 1, dtype=dtype, device="cuda"), 0 * one, one, out, one, one, out)
    assert out.item() == -5
    ops.check_errors()
