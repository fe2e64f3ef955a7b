"""What a profiler sees of the serving operators: an event of each call, with the shapes of its inputs."""

import pytest
import torch
from torch.profiler import ProfilerActivity, profile

import numa_allreduce_b200 as nab

BF = torch.bfloat16


def events(call, record_shapes=True):
    with profile(activities=[ProfilerActivity.CPU], record_shapes=record_shapes) as p:
        with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
            call()
    return {e.name: e.input_shapes for e in p.events() if e.name.startswith("nab::")}


def test_shapes_are_recorded():
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    pages = torch.zeros(3, 2, 16, 64, dtype=BF), torch.zeros(3, 2, 16, 64, dtype=BF)
    got = events(lambda: nab.assign_pages(i32(2), i32(2, 4), i32(3), i32(1), 16))
    assert [s for s in got["nab::assign_pages"] if s] == [[2], [2, 4], [3], [1]]
    got = events(lambda: nab.rope_append_paged(torch.zeros(5, 512, dtype=BF), torch.zeros(9, 32), torch.zeros(9, 32),
                                               i32(5), torch.arange(5), *pages, 4, k_norm=torch.ones(64, dtype=BF)))
    assert [s for s in got["nab::rope_append_paged"] if s] == [[5, 512], [9, 32], [9, 32], [5], [5], [3, 2, 16, 64],
                                                               [3, 2, 16, 64], [64]]
    got = events(lambda: nab.paged_attention(torch.zeros(2, 4, 64, dtype=BF), *pages, i32(2, 3), i32(2)))
    assert [s for s in got["nab::paged_attention"] if s] == [[2, 4, 64], [3, 2, 16, 64], [3, 2, 16, 64], [2, 3], [2]]
    got = events(lambda: nab.token_logprobs(torch.zeros(2, 10), torch.zeros(2, dtype=torch.long), top_k=3))
    assert [s for s in got["nab::token_logprobs"] if s] == [[2, 10], [2]]
    assert "nab::token_logprobs" in events(
        lambda: nab.token_logprobs(torch.zeros(2, 10), torch.zeros(2, dtype=torch.long)), record_shapes=False)
