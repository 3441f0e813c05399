"""What the operators of an 8-bit cache tell their kernels, read from the packed arguments; no kernel runs."""
import pytest
import torch

from pytriton_llama_b200.ops.cuda import CudaOps, KernelError

I32, BF = torch.int32, torch.bfloat16


class Library:
    """Keeps what an entry was called with."""

    def __init__(self):
        self.calls = {}

    def __getattr__(self, name):
        def entry(packed):
            self.calls[name] = packed
            return 0
        return entry


@pytest.fixture()
def ops():
    o = CudaOps.__new__(CudaOps)
    o.device, o.lib, o._raw_stream, o._device_index, o.launches, o._sm_count = torch.device("cpu"), Library(), lambda i: 0, 0, 0, 148
    o._tc_status_word = lambda: torch.zeros(1, dtype=I32)
    return o


def test_integers_are_read_early_inside_of_a_forward_pass_only(ops):
    """There the step's integers came before its first kernel; elsewhere they may come from the kernel before."""
    codes, words = torch.zeros((9, 2, 2, 16, 64), dtype=torch.uint8), torch.zeros((9, 2, 1, 2), dtype=I32)

    def early():
        ops.lib.calls.clear()
        ops.rope_kv8_write(torch.zeros((3, 512), dtype=BF), torch.zeros(3, dtype=I32), torch.zeros(32), 64, torch.zeros(3, dtype=I32), codes, words, 4, 2, 64, 16)
        write = int("ptl_rope_kv8_write_early_bf16" in ops.lib.calls)
        hints = ops.hints_for([20], [100])
        hints.split_portions = False
        ops.paged_attention8(torch.zeros((20, 256), dtype=BF), codes, words, torch.zeros((1, 7), dtype=I32), torch.zeros(20, dtype=I32),
                             torch.arange(80, 100, dtype=I32), 4, 2, 64, 16, 0.125, hints=hints)
        return write, ops._PREFILL8_ARGS.unpack(ops.lib.calls["ptl_attention8_prefill_tc_bf16"])[-1]
    assert early() == (0, 0)
    ops.begin_forward()
    assert early() == (1, 1)
    ops.end_forward()
    assert early() == (0, 0)


def attend(ops, tokens, q_lens, requests=2, **forms):
    codes, words = torch.zeros((9, 2, 2, 16, 64), dtype=torch.uint8), torch.zeros((9, 2, 1, 2), dtype=I32)
    hints = ops.hints_for(q_lens, [n + 30 for n in q_lens])
    for name, value in forms.items():
        setattr(hints, name, value)
    return ops.paged_attention8(torch.zeros((tokens, 256), dtype=BF), codes, words, torch.zeros((requests, 4), dtype=I32), torch.zeros(tokens, dtype=I32),
                                torch.zeros(tokens, dtype=I32), 4, 2, 64, 16, 0.125, hints=hints)


@pytest.mark.parametrize("q_lens,requests", [([1, 4], 2), ([6], 2), ([1, 1, 1], 2)])
def test_lists_of_more_rows_or_requests_than_there_are_are_refused(ops, q_lens, requests):
    """The kernels go by the lists: they would write behind the output, or read behind the table."""
    with pytest.raises(KernelError, match="the step's lists are of"):
        attend(ops, 4, q_lens, requests)
    assert not ops.lib.calls


def test_rows_behind_those_of_the_lists_are_zeros(ops):
    """No kernel writes them; those of a captured step's padding are nobody's."""
    ops.lib.calls["ptl_attention8_units"] = None
    torch.utils.deterministic.fill_uninitialized_memory, was = True, torch.are_deterministic_algorithms_enabled()
    torch.use_deterministic_algorithms(True)               # (memory that is not written is NaN)
    try:
        for q_lens in ([3], [1, 4], [1, 1], [40]):
            T = sum(q_lens)
            assert torch.isnan(attend(ops, T, q_lens, single_form=(1, 4)).float()).all()
            assert not attend(ops, T + 3, q_lens, single_form=(1, 4))[T:].any()
            assert torch.isnan(attend(ops, T + 3, q_lens, single_form=(1, 4), host_lengths_exact=False).float()).all()
    finally:
        torch.use_deterministic_algorithms(was)
