"""A paged decoder whose requests run out of pages says so under NAB_CHECK=1
(on the CPU, with stand-ins for the CUDA kernels)."""

import pytest
import torch

import numa_allreduce_b200 as nab
from numa_allreduce_b200.models import llama_tp
from test_decoder_choice_cpu import decoder, stand_ins


@pytest.fixture
def full(monkeypatch):
    """A decoder with one request that has no page left for its next token."""
    stand_ins(monkeypatch.setattr)
    monkeypatch.setattr(llama_tp, "check_kernels", lambda: None)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)

    def assign(cached, tables, free, taken, page):
        lengths = cached + 1
        lengths[2] = torch.minimum(lengths[2], torch.tensor(4, dtype=lengths.dtype))
        return nab.PageSlots(cached, cached.long(), lengths, taken)

    monkeypatch.setattr(llama_tp, "assign_pages", assign)
    return decoder(256)


def test_a_token_without_a_page_is_an_error_on_request(full, monkeypatch):
    monkeypatch.setenv("NAB_CHECK", "1")
    full.step()  # to 4 positions
    full.advance()
    with pytest.raises(nab.KernelError, match=r"no page.*requests \[2\]"):
        full.step()


def test_and_goes_on_without_the_request(full, monkeypatch):
    monkeypatch.delenv("NAB_CHECK", raising=False)
    for _ in range(3):
        full.step()
        full.advance()
    assert full.cached.tolist() == [6, 6, 4, 6, 6, 6]
