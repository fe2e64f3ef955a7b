"""The token that a decode step chooses, on the CPU: the decoder's own step and
advance, with stand-ins for the CUDA kernels, on one rank and over gloo ranks.

The output weight of every rank is padded to a multiple of 128 columns; the
columns past the vocabulary hold weights like any others and must never be
chosen, or the next step reads past the embedding.
"""

import types

import pytest
import torch
import torch.distributed as dist
import torch.nn.functional as F

import numa_allreduce_b200 as nab
from numa_allreduce_b200.models import llama_tp
from numa_allreduce_b200.models.llama_tp import LlamaConfig, LlamaTPDecoder


def config(vocab):
    return LlamaConfig(hidden=64, layers=1, heads=4, kv_heads=4, head_dim=64, intermediate=128, vocab=vocab)


def _logprobs(logits, tokens, top_k=0, vocab_start=0):
    x = logits.double()
    lse = x.logsumexp(-1)
    lp = x - lse[:, None]
    at = tokens - vocab_start
    inside = (at >= 0) & (at < x.shape[1])
    picked = torch.where(inside, lp.gather(1, torch.where(inside, at, 0)[:, None])[:, 0], -torch.inf)
    order = x.argsort(dim=-1, descending=True, stable=True)[:, :top_k]
    return nab.TokenLogprobs(picked, -(lp.exp() * lp).sum(-1), lse, lp.gather(1, order), order + vocab_start,
                             x.gather(1, order))


def stand_ins(setattr_):
    """CPU forms of the kernels of a baseline step over pages; the attention gives back its queries."""
    setattr_(llama_tp, "assign_pages", lambda cached, tables, free, taken, page:
             nab.PageSlots(cached, cached.long(), cached + 1, taken))
    setattr_(llama_tp, "rope_append_paged", lambda qkv, *a, out: out.copy_(qkv[:, :out[0].numel()].view_as(out)))
    setattr_(llama_tp, "paged_attention", lambda q, *a, out: out.copy_(q))
    setattr_(llama_tp, "token_logprobs", _logprobs)


def decoder(vocab, comm=None, **kw):
    m = LlamaTPDecoder(config(vocab), comm, batch=6, context=3, impl="baseline", device="cpu", kv="paged", max_new=9,
                       **kw)
    m.ops = types.SimpleNamespace(silu_mul=lambda gu, act: act.copy_(F.silu(gu[:, :m.I]) * gu[:, m.I:]))
    m.lm_head[max(0, m.v_valid):] *= 50  # padding columns win any comparison
    return m


@pytest.mark.parametrize("vocab", [1, 100, 256, 300])
def test_a_step_chooses_within_the_vocabulary(vocab, monkeypatch):
    stand_ins(monkeypatch.setattr)
    m = decoder(vocab, logprobs=1)
    for _ in range(4):
        assert (m.tokens < vocab).all()
        m.step()
        valid = m.logits[:, :vocab].float()
        assert torch.equal(valid.gather(1, m.next_tokens[:, None])[:, 0], valid.amax(-1))
        assert torch.equal(m.logprobs.logprob, m.logprobs.top_logprobs[:, 0])  # the best one, and it has a probability
        m.advance()


def _rank(rank, world, port, path, vocab):
    dist.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{port}", rank=rank, world_size=world)
    stand_ins(setattr)
    comm = types.SimpleNamespace(world_size=world, rank=rank, disabled=False)
    share = vocab - (world - 1) * (((vocab + world - 1) // world + 127) // 128 * 128)
    m = decoder(vocab, comm, logprobs=2 if share >= 2 else None)
    chosen = []
    for _ in range(4):
        m.step()
        logits = torch.empty(world, 6, m.v_local, dtype=m.logits.dtype)
        dist.all_gather(list(logits.unbind(0)), m.logits)
        chosen.append((m.next_tokens.clone(), logits.transpose(0, 1).reshape(6, -1)[:, :vocab].float(), m.logprobs))
        m.advance()
    torch.save(chosen, f"{path}/{rank}.pt")
    dist.barrier()
    dist.destroy_process_group()


# 4 ranks x 128 columns: 12 columns on the last one, and none on the last two
@pytest.mark.parametrize("world,vocab", [(2, 300), (4, 396), (4, 200)])
def test_ranks_choose_within_the_vocabulary(world, vocab, tmp_path):
    import torch.multiprocessing as mp

    from conftest import free_port

    mp.spawn(_rank, args=(world, free_port(), str(tmp_path), vocab), nprocs=world)
    for rank in range(world):
        for tokens, logits, logprobs in torch.load(tmp_path / f"{rank}.pt", weights_only=False):
            assert (tokens < vocab).all()
            assert torch.equal(logits.gather(1, tokens[:, None])[:, 0], logits.amax(-1))
            if logprobs is not None:
                assert torch.equal(logprobs.top_logits[:, 0].float(), logits.amax(-1))
                # float64 throughout
                torch.testing.assert_close(logprobs.logprob, logprobs.top_logprobs[:, 0], rtol=0, atol=1e-13)


@pytest.mark.parametrize("rank", range(4))
def test_every_rank_refuses_more_alternatives_than_the_last_one_has(rank):
    comm = types.SimpleNamespace(world_size=4, rank=rank, disabled=False)
    with pytest.raises(ValueError, match="vocabulary"):
        decoder(396, comm, logprobs=13)
    with pytest.raises(ValueError, match="vocabulary"):
        decoder(200, comm, logprobs=0)  # the last two have no column at all
