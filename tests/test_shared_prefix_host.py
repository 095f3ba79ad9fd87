"""What `CudaOps.shared_prefix_attention` refuses before it launches anything, without a GPU."""

import ctypes

import pytest
import torch

from somi_inference_b200.ops import KernelError, cuda


class OnDevice(torch.Tensor):
    """A CPU tensor that the host side takes for one of device 0's."""
    is_cuda = True

    def get_device(self):
        return 0


def on_device(t):
    return t.as_subclass(OnDevice)


@pytest.fixture
def ops(monkeypatch):
    """A kernel table over CPU tensors whose launcher notes its calls."""
    table = cuda.CudaOps.__new__(cuda.CudaOps)
    table.launches, table._device_index, table.calls = 0, 0, []
    table._shared_plans, table.use_shared_tc = {}, True
    table.lib = type("Library", (), {})()
    table.lib.somi_shared_attention_ctas = lambda hd, kernel: 148
    table.lib.somi_shared_attention_block_rows = lambda kernel: 64
    table._shared_attention = lambda *a: table.calls.append(a) or 0
    table._stream = lambda: ctypes.c_void_p(0)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    return table


def arguments(**changed):
    T, R, G, nq, nkv, hd, page = 3, 3, 1, 4, 2, 64, 16
    a = dict(qkv=torch.zeros(T, nq * hd), kcache=torch.zeros(9, nkv, page, hd), vcache=torch.zeros(9, nkv, page, hd),
             block_table=torch.zeros(R, 5, dtype=torch.int32), ctx_len=torch.zeros(R, dtype=torch.int32),
             prefix_len=torch.zeros(G, dtype=torch.int32), group_off=torch.zeros(G + 1, dtype=torch.int32),
             nq=nq, nkv=nkv, hd=hd, scale=1.0, out=torch.zeros(T, nq * hd), cu_q=None)
    a.update(changed)
    return {n: on_device(t) if isinstance(t, torch.Tensor) else t for n, t in a.items()}


def test_a_consistent_call_launches_with_a_workspace_that_holds_all_parts(ops):
    ops.shared_prefix_attention(**arguments())
    (call,) = ops.calls
    rows = 2 * 3 * 4 + 148 * 64
    assert call[-4] == 32 * 3 + 32 + rows * (8 + 4 * 64) and call[-3] == 148 and ops.launches == 2


@pytest.mark.parametrize("changed", [
    dict(out=torch.zeros(3, 128)),
    dict(out=torch.zeros(3, 256, dtype=torch.bfloat16)),
    dict(qkv=torch.zeros(3, 255)),
    dict(qkv=torch.zeros(3, 512)[:, ::2]),
    dict(qkv=torch.zeros(3, 257)[:, :256]),                        # rows not on 16-byte boundaries
    dict(qkv=torch.zeros(3 * 256 + 1)[1:].view(3, 256)),
    dict(kcache=torch.zeros(9, 2, 16, 64).bfloat16()),
    dict(vcache=torch.zeros(8, 2, 16, 64)),
    dict(kcache=torch.zeros(9, 1, 16, 64), vcache=torch.zeros(9, 1, 16, 64)),
    dict(kcache=torch.zeros(9, 2, 64, 16).transpose(2, 3)),
    dict(block_table=torch.zeros(2, 5, dtype=torch.int32)),
    dict(block_table=torch.zeros(3, 5, dtype=torch.int64)),
    dict(ctx_len=torch.zeros(3)),
    dict(group_off=torch.zeros(1, dtype=torch.int32)),
    dict(cu_q=torch.zeros(3, dtype=torch.int32)),
    dict(qkv=torch.zeros(4, 256), out=torch.zeros(4, 256)),        # one token per request, and four tokens
    dict(hd=24, qkv=torch.zeros(3, 96), out=torch.zeros(3, 96), kcache=torch.zeros(9, 2, 16, 24), vcache=torch.zeros(9, 2, 16, 24)),
    dict(nq=3, qkv=torch.zeros(3, 192), out=torch.zeros(3, 192)),
])
def test_refusals(ops, changed):
    with pytest.raises(KernelError):
        ops.shared_prefix_attention(**arguments(**changed))
    assert not ops.calls and ops.launches == 0


def test_a_tensor_of_the_host_or_another_device_is_refused(ops):
    a = arguments()
    a["ctx_len"] = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(KernelError):
        ops.shared_prefix_attention(**a)
    ops._device_index = 1
    with pytest.raises(KernelError, match="device"):
        ops.shared_prefix_attention(**arguments())
    assert not ops.calls


def test_what_the_launcher_refuses_is_an_error(ops):
    ops._shared_attention = lambda *a: cuda.ERR_UNSUPPORTED
    with pytest.raises(KernelError, match="not supported"):
        ops.shared_prefix_attention(**arguments())


def test_the_rule_of_a_step(ops):
    """Which steps of forked requests go the shared way: by type, head sizes and what it saves."""
    from types import SimpleNamespace
    ops.use_shared_prefix = True
    ops.lib.somi_shared_attention_tc_takes = lambda nq, nkv, hd, page: int(hd in (64, 128) and 128 % page == 0)
    rows = {d: torch.zeros(2, 36 * 128, dtype=d) for d in (torch.bfloat16, torch.float32)}

    def pays(saved, singles=0, portions=0, tokens=0, dtype=torch.bfloat16, page=16, hd=128, qkv=None):
        batch = SimpleNamespace(num_requests=singles + portions, num_prefill_requests=portions, num_prefill_tokens=tokens,
                                num_tokens=singles + tokens)
        return ops.shared_prefix_pays(saved.bit_length(), batch, 28, 4, hd, rows[dtype] if qkv is None else qkv, page)

    assert pays(63 * 2048, 64) and pays(7 * 8192, 8) and not pays(7 * 2048, 8) and not pays(63 * 512, 64)
    assert not pays(15 * 4096, 80) and pays(15 * 4096, 40)         # beside many that share nothing
    assert not pays(63 * 2048, 64, dtype=torch.float32) and not pays(63 * 2048, 64, page=24) and not pays(63 * 2048, 64, hd=96)
    assert not pays(63 * 2048, 64, qkv=rows[torch.bfloat16][:, :-4]) and not pays(10 ** 9, 5000)
    assert pays(3 * 2048, 0, 4, 64) and not pays(15 * 64, 0, 16, 64) and pays(15 * 4096, 0, 16, 16 * 64)
    assert not pays(15 * 176, 0, 16, 16 * 64) and not pays(15 * 4096, 0, 16, 16 * 200)
    ops.use_shared_prefix = False
    assert not pays(63 * 2048, 64)


def test_the_rule_of_a_step_of_portions_and_single_tokens(ops):
    """Portions that share nothing leave the decision to the single tokens, unless they lie behind many positions of their
    own; requests that share nothing, and long portions, count against what is saved."""
    from types import SimpleNamespace
    from somi_inference_b200.engine.batch import PortionFacts
    ops.use_shared_prefix = True
    ops.lib.somi_shared_attention_tc_takes = lambda nq, nkv, hd, page: 1

    def pays(saved, portions, singles=0, by_portions=0, deep=False, long=False, heads=(28, 4, 128)):
        """`portions`: their tokens."""
        nq, nkv, hd = heads
        batch = SimpleNamespace(num_requests=singles + len(portions), num_prefill_requests=len(portions),
                                num_prefill_tokens=sum(portions), num_tokens=singles + sum(portions))
        facts = PortionFacts(by_portions.bit_length(), deep, long)
        return ops.shared_prefix_pays(saved.bit_length(), batch, nq, nkv, hd, torch.zeros(1, (nq + 2 * nkv) * hd).bfloat16(), 16, facts)

    # single tokens that are refused alone are refused beside a prompt that shares nothing
    assert not pays(7 * 2048, [16], singles=8) and not pays(7 * 512, [2], singles=8) and not pays(1024, [16], singles=2)
    assert pays(7 * 2048, [16], singles=8, deep=True) and not pays(7 * 2048, [16], singles=108, deep=True)
    # ... and those that are taken alone are taken, if it is short
    assert pays(15 * 4096, [16], singles=16) and not pays(15 * 4096, [300], singles=16) and not pays(15 * 4096, [16], singles=80)
    # portions that share
    assert pays(1024, [16, 16], by_portions=1024) and pays(1024, [16, 16], singles=64, by_portions=1024)
    assert not pays(1024, [16, 16], singles=200, by_portions=1024) and not pays(3 * 512, [2] * 4, singles=200, by_portions=3 * 512)
    # what portions save among themselves is too little, and the single tokens decide
    assert not pays(7 * 2048 + 16, [2, 2], singles=8, by_portions=16)
    # thirty of 2 beside one of 900, and beside one of 1,025
    assert pays(29 * 2048, [2] * 30 + [900], by_portions=29 * 2048)
    assert not pays(29 * 2048, [2] * 60 + [1025], by_portions=29 * 2048, long=True)
    # few elements a position: more positions a request
    small = (14, 2, 64)
    assert pays(63 * 8192, [], singles=64, heads=small) and not pays(39 * 4096, [], singles=148, heads=small)
    assert pays(39 * 4096, [], singles=148) and not pays(0, [16, 16], singles=4)


def test_the_kernel_that_scales_a_maximum_takes_positive_scales_only(ops):
    ops.lib.somi_shared_attention_tc_takes = lambda nq, nkv, hd, page: 1
    many = {n: torch.zeros(40, 5, dtype=torch.int32) if n == "block_table" else torch.zeros(40, dtype=torch.int32)
            for n in ("block_table", "ctx_len")}
    many.update({n: torch.zeros(40, 256).bfloat16() for n in ("qkv", "out")})
    many.update({n: torch.zeros(9, 2, 16, 64).bfloat16() for n in ("kcache", "vcache")})
    for scale, kernel in ((0.5, 1), (-0.5, 0), (0.5, 1), (0.0, 0), (float("nan"), 0)):
        ops.shared_prefix_attention(**arguments(scale=scale, **many))
        assert ops.calls[-1][20] == kernel
