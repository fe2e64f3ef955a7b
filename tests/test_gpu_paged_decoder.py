"""LlamaTPDecoder over a paged cache on one GPU: against the contiguous cache
with the same weights and contents, token after token, and its
log-probabilities."""

import math

import pytest
import torch

import numa_allreduce_b200 as nab
from numa_allreduce_b200.models.llama_tp import LlamaConfig, LlamaTPDecoder

pytestmark = pytest.mark.gpu


def share_weights(a, b):
    """b's layers take a's weights (before either packs them)."""
    for x, y in zip(a.layers, b.layers):
        for k in ("wqkv", "wo", "wgu", "wd", "in_norm", "post_norm"):
            y[k] = x[k]
    b.embed, b.lm_head, b.final_norm = a.embed, a.lm_head, a.final_norm


def copy_cache(paged, flat, request, row):
    """Row `row` of flat's contiguous cache := request `request` of the pages."""
    n = int(paged.cached[request])
    ids = paged.block_tables[request, :-(-n // paged.page_size)].long()
    for x, y in zip(paged.layers, flat.layers):
        for k in ("k", "v"):
            y[k][row, :, :n] = x[k][ids].transpose(0, 1).reshape(paged.Hkv, -1, 128)[:, :n]


@pytest.mark.parametrize("impl", ["fused", "baseline"])
@pytest.mark.parametrize("lengths,page", [([100, 100, 100], 64), ([3, 129, 64, 0, 257], 16), ([1024], 128)])
def test_paged_step_matches_the_contiguous_cache(lengths, page, impl):
    cfg = LlamaConfig.tiny()
    m = LlamaTPDecoder(cfg, None, batch=len(lengths), context=0, kv="paged", lengths=lengths, page_size=page, impl=impl)
    m.tokens.copy_(torch.arange(len(lengths), device="cuda") * 11 + 5)
    flats = []
    for i, n in enumerate(lengths):
        f = LlamaTPDecoder(cfg, None, batch=1, context=n, impl=impl)
        share_weights(m, f)
        copy_cache(m, f, i, 0)
        f.tokens.copy_(m.tokens[i:i + 1])
        flats.append(f)
    m.step()
    for i, f in enumerate(flats):
        f.step()
        # two bf16 paths that differ in the order of sums only: the margin of the decoder's other tests
        rel = ((m.x[i].float() - f.x[0].float()).norm() / f.x[0].float().norm()).item()
        assert rel < 2e-2, (i, rel)
    assert m.paged_step.lengths.tolist() == [n + 1 for n in lengths]
    nab.check_kernels()


def test_decoding_token_after_token():
    """Eager steps, and one captured step + advance replayed: the same tokens, lengths, pages and caches."""
    cfg = LlamaConfig.tiny()
    lengths, steps = [14, 0, 31, 100], 40
    runs = []
    for capture in (False, True):
        m = LlamaTPDecoder(cfg, None, batch=4, context=0, kv="paged", lengths=lengths, page_size=16, max_new=steps,
                           logprobs=3)
        m.tokens.copy_(torch.tensor([1, 2, 3, 4], device="cuda"))
        got = []
        if capture:
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                m.step()
            torch.cuda.current_stream().wait_stream(s)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                m.step()
                m.advance()
        for _ in range(steps):
            if capture:
                g.replay()
            else:
                m.step()
                m.advance()
            got.append((m.tokens.tolist(), m.cached.tolist(), m.taken.tolist(), m.logprobs.top_tokens.tolist()))
        assert m.cached.tolist() == [n + steps for n in lengths]
        assert m.taken.item() == m.free_pages.numel()
        runs.append((got, m.block_tables.tolist(), [L["k"].clone() for L in m.layers]))
        m.reset_position()
        assert m.cached.tolist() == lengths and m.taken.item() == 0
        if capture:
            del g
    assert runs[0][0] == runs[1][0] and runs[0][1] == runs[1][1]
    for a, b in zip(runs[0][2], runs[1][2]):
        assert torch.equal(a, b)
    nab.check_kernels()


@pytest.mark.parametrize("kv", ["contiguous", "paged"])
def test_logprobs_of_a_step(kv):
    cfg = LlamaConfig.tiny()
    m = LlamaTPDecoder(cfg, None, batch=3, context=70, kv=kv, logprobs=5)
    m.tokens.copy_(torch.tensor([7, 8, 9], device="cuda"))
    m.step()
    lp = m.logits.double()[:, :cfg.vocab].log_softmax(-1)
    r = m.logprobs
    # fp32 sums over 4096 bf16 logits of a few units: within 2^-16 (64 + 8 roundings of 2^-23, values below 16)
    assert (r.logprob.double() - lp.gather(1, m.next_tokens[:, None])[:, 0]).abs().max() < 2 ** -16
    assert (r.entropy.double() + (lp.exp() * lp).sum(-1)).abs().max() < 2 ** -15
    values, ids = m.logits.double()[:, :cfg.vocab].sort(dim=-1, descending=True, stable=True)
    assert torch.equal(r.top_tokens, ids[:, :5])
    assert torch.equal(r.top_logits.double(), values[:, :5])


def test_a_full_pool_stops_growing():
    """Past max_new the requests keep their length; nothing is written outside the pool."""
    cfg = LlamaConfig.tiny()
    m = LlamaTPDecoder(cfg, None, batch=2, context=0, kv="paged", lengths=[15, 16], page_size=16, max_new=1)
    m.tokens.copy_(torch.tensor([1, 2], device="cuda"))
    for _ in range(20):
        m.step()
        m.advance()
    assert m.cached.tolist() == [16, 32]
    nab.check_kernels()
    assert math.isfinite(m.x.float().sum().item())
