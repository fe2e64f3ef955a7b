"""Refusals of the paged-cache operators and the token log-probabilities, the
rotary tables and the join of vocabulary shards: what needs no GPU."""

import math

import pytest
import torch

import numa_allreduce_b200 as nab
from numa_allreduce_b200.ops import _ext


def _i32(*v):
    return torch.tensor(v, dtype=torch.int32)


def _assign(**kw):
    a = dict(cached=_i32(3, 20), block_tables=torch.zeros(2, 4, dtype=torch.int32), free_pages=_i32(4, 5, 6),
             taken=_i32(0), page_size=16)
    a.update(kw)
    return nab.assign_pages(**a)


@pytest.mark.parametrize("kw,match", [
    (dict(cached=torch.zeros(0, dtype=torch.int32)), "1 to 8192 requests"),
    (dict(cached=torch.zeros(8193, dtype=torch.int32)), "1 to 8192 requests"),
    (dict(cached=torch.zeros(2, dtype=torch.int64)), "cached"),
    (dict(cached=torch.zeros(2, 2, dtype=torch.int32)[:, 0]), "cached"),
    (dict(block_tables=torch.zeros(3, 4, dtype=torch.int32)), "block_tables"),
    (dict(block_tables=torch.zeros(2, 4)), "block_tables"),
    (dict(block_tables=torch.zeros(1, 4, dtype=torch.int32).expand(2, 4)), "apart"),
    (dict(block_tables=torch.zeros(4, 2, dtype=torch.int32).t()), "contiguous"),
    (dict(free_pages=torch.zeros(3)), "free_pages"),
    (dict(free_pages=torch.zeros(6, dtype=torch.int32)[::2]), "free_pages"),
    (dict(taken=_i32(0, 1)), "taken"),
    (dict(page_size=0), "page_size"),
    (dict(page_size=24), "page_size"),
    (dict(query_start=_i32(0, 1), num_tokens=2), "query_start"),
    (dict(num_tokens=1), "num_tokens"),
    (dict(query_start=_i32(0, 1, 2), num_tokens=-1), "num_tokens"),
    (dict(), "must be a CUDA tensor"),
])
def test_assign_pages_refuses(kw, match):
    with pytest.raises(RuntimeError, match=match):
        _assign(**kw)


def test_assign_pages_needs_the_row_count_of_a_ragged_step():
    with pytest.raises(ValueError, match="num_tokens"):
        _assign(query_start=_i32(0, 1, 2))


def _append(**kw):
    bf = torch.bfloat16
    a = dict(qkv=torch.zeros(3, 8 * 64, dtype=bf), cos=torch.zeros(10, 32), sin=torch.zeros(10, 32),
             positions=torch.zeros(3, dtype=torch.int32), slots=torch.arange(3),
             k_pages=torch.zeros(2, 2, 16, 64, dtype=bf), v_pages=torch.zeros(2, 2, 16, 64, dtype=bf), q_heads=4)
    a.update(kw)
    return nab.rope_append_paged(**a)


BF = torch.bfloat16


@pytest.mark.parametrize("kw,match", [
    (dict(qkv=torch.zeros(3, 512)), "qkv must be bfloat16 or float16"),
    (dict(qkv=torch.zeros(3, 511, dtype=BF)), "qkv"),
    (dict(qkv=torch.zeros(512, 3, dtype=BF).t()), "contiguous rows"),
    (dict(qkv=torch.zeros(3, 516, dtype=BF)[:, :512]), "16-byte aligned"),
    (dict(qkv=torch.zeros(3, 520, dtype=BF)[:, 4:516]), "16-byte aligned"),
    (dict(k_pages=torch.zeros(2, 2, 16, 64)), "k_pages"),
    (dict(k_pages=torch.zeros(2, 16, 2, 64, dtype=BF).transpose(1, 2)), "contiguous"),
    (dict(v_pages=torch.zeros(3, 2, 16, 64, dtype=BF)), "one shape"),
    (dict(k_pages=torch.zeros(2, 2, 24, 64, dtype=BF), v_pages=torch.zeros(2, 2, 24, 64, dtype=BF)), "page_size"),
    (dict(k_pages=torch.zeros(2, 2, 8, 64, dtype=BF), v_pages=torch.zeros(2, 2, 8, 64, dtype=BF)), "page_size"),
    (dict(k_pages=torch.zeros(2, 2, 16, 96, dtype=BF), v_pages=torch.zeros(2, 2, 16, 96, dtype=BF)), "head_dim"),
    (dict(k_pages=torch.zeros(0, 2, 16, 64, dtype=BF), v_pages=torch.zeros(0, 2, 16, 64, dtype=BF)), "no pages"),
    (dict(cos=torch.zeros(10, 20), sin=torch.zeros(10, 20)), "rotary_dim"),
    (dict(cos=torch.zeros(10, 40), sin=torch.zeros(10, 40)), "rotary_dim"),
    (dict(sin=torch.zeros(9, 32)), "cos and sin"),
    (dict(cos=torch.zeros(10, 32, dtype=BF)), "cos and sin"),
    (dict(positions=torch.zeros(3, dtype=torch.int64)), "positions"),
    (dict(slots=torch.zeros(3, dtype=torch.int32)), "slots"),
    (dict(slots=torch.zeros(2, dtype=torch.int64)), "slots"),
    (dict(q_norm=torch.ones(64)), "q_norm"),
    (dict(k_norm=torch.ones(32, dtype=BF)), "k_norm"),
    (dict(q_heads=5, qkv=torch.zeros(3, 9 * 64, dtype=BF)), "do not divide"),
    (dict(out=torch.zeros(3, 4, 64)), "out"),
    (dict(out=torch.zeros(3, 2, 64, dtype=BF)), "out"),
    (dict(out=torch.zeros(3, 4, 128, dtype=BF)[..., ::2]), "out"),
    (dict(q_heads=0, qkv=torch.zeros(3, 4 * 64, dtype=BF)), "do not divide"),
    (dict(qkv=torch.zeros(3, 512, dtype=BF, requires_grad=True)), "requires a gradient"),
    (dict(), "must be a CUDA tensor"),
])
def test_rope_append_paged_refuses(kw, match):
    with pytest.raises(RuntimeError, match=match):
        _append(**kw)


def _attend(**kw):
    a = dict(q=torch.zeros(2, 4, 64, dtype=BF), k_pages=torch.zeros(3, 2, 16, 64, dtype=BF),
             v_pages=torch.zeros(3, 2, 16, 64, dtype=BF), block_tables=torch.zeros(2, 3, dtype=torch.int32),
             lengths=_i32(4, 5))
    a.update(kw)
    return nab.paged_attention(**a)


@pytest.mark.parametrize("kw,match", [
    (dict(q=torch.zeros(2, 4, 64)), "q must be bfloat16 or float16"),
    (dict(q=torch.zeros(2, 4, 64, dtype=torch.float16)), "k_pages and v_pages must be"),
    (dict(q=torch.zeros(2, 4, 128, dtype=BF)), "q must be"),
    (dict(q=torch.zeros(2, 3, 64, dtype=BF)), "do not divide"),
    (dict(q=torch.zeros(4, 2, 64, dtype=BF).transpose(0, 1)), "q must be contiguous|heads of q"),
    (dict(q=torch.zeros(2, 288, dtype=BF)[:, :256].view(2, 4, 64)), "multiple of head_dim apart"),
    (dict(q=torch.zeros(1, 4, 64, dtype=BF).expand(2, 4, 64)), "heads of q"),
    (dict(out=torch.zeros(2, 4, 64)), "out"),
    (dict(out=torch.zeros(2, 8, 64, dtype=BF)[:, ::2]), "out"),
    (dict(block_tables=torch.zeros(2, 3, dtype=torch.int64)), "block_tables"),
    (dict(block_tables=torch.zeros(3, 2, dtype=torch.int32).t()), "contiguous rows"),
    (dict(lengths=torch.zeros(2, dtype=torch.int64)), "lengths"),
    (dict(lengths=_i32(1, 2, 3)), "lengths"),
    (dict(q=torch.zeros(2, 4, 64, dtype=BF, requires_grad=True)), "requires a gradient"),
    (dict(), "must be a CUDA tensor"),
])
def test_paged_attention_refuses(kw, match):
    with pytest.raises(RuntimeError, match=match):
        _attend(**kw)


@pytest.mark.parametrize("kw,match", [
    (dict(logits=torch.zeros(2, 10, dtype=torch.float64)), "logits must be float32"),
    (dict(logits=torch.zeros(10)), "logits must be"),
    (dict(logits=torch.zeros(10, 2).t()), "contiguous rows"),
    (dict(logits=torch.zeros(2, 0)), "logits must be"),
    (dict(tokens=torch.zeros(2, dtype=torch.int32)), "tokens"),
    (dict(tokens=torch.zeros(3, dtype=torch.int64)), "tokens"),
    (dict(top_k=11), "top_k"),
    (dict(top_k=-1), "top_k"),
    (dict(logits=torch.zeros(2, 100), top_k=33), "top_k"),
    (dict(vocab_start=-1), "vocab_start"),
    (dict(logits=torch.zeros(2, 10, requires_grad=True)), "requires a gradient"),
    (dict(), "must be a CUDA tensor"),
])
def test_token_logprobs_refuses(kw, match):
    a = dict(logits=torch.zeros(2, 10), tokens=torch.zeros(2, dtype=torch.int64), top_k=3)
    a.update(kw)
    with pytest.raises(RuntimeError, match=match):
        nab.token_logprobs(**a)


def test_an_index_out_of_range_is_named(monkeypatch):
    from numa_allreduce_b200.ops import errors

    class Ops:
        def kernel_error_code(self):
            return 2

        def kernel_error_state(self):
            return [2, 0xFFFFFFFF, 0xFFFFFFFF, 13, 5, 0, 77, 3]

    monkeypatch.setattr(errors._ext, "load", lambda: Ops())
    with pytest.raises(errors.KernelError, match="index out of range.*value 77, 3 of them"):
        errors.check_kernels(sync=False)


# ------------------------------------------------------------ rotary tables --
def test_rope_tables_plain():
    cos, sin = nab.rope_tables(50, 32, theta=500000.0, device="cpu")
    assert cos.shape == sin.shape == (50, 16) and cos.dtype == torch.float32
    for p, i in ((0, 0), (1, 0), (49, 3), (37, 15)):
        ang = p * 500000.0 ** (-2 * i / 32)
        # one rounding to float32
        assert abs(cos[p, i].item() - math.cos(ang)) <= 2 ** -24 and abs(sin[p, i].item() - math.sin(ang)) <= 2 ** -24


def test_rope_tables_scaled():
    base = nab.rope_tables(9, 32, theta=1e4, device="cpu")
    far = nab.rope_tables(33, 32, theta=1e4, scale=4.0, device="cpu")
    # every frequency divided by 4: position 4p has the angle of p
    torch.testing.assert_close(far[0][::4], base[0], rtol=0, atol=2 ** -22)
    ramp = nab.rope_tables(33, 32, theta=1e4, scale=4.0, original_positions=512, low=1.0, high=4.0, device="cpu")
    for i in range(16):
        f = 1e4 ** (-2 * i / 32)
        wave = 2 * math.pi / f
        if wave < 512 / 4:
            want = f
        elif wave > 512:
            want = f / 4
        else:
            s = (512 / wave - 1) / 3
            want = (1 - s) * f / 4 + s * f
        assert abs(ramp[1][32, i].item() - math.sin(32 * want)) <= 2 ** -23


@pytest.mark.parametrize("kw", [dict(max_positions=0), dict(rotary_dim=3), dict(scale=0.0), dict(theta=-1.0),
                                dict(original_positions=100, low=2.0, high=1.0)])
def test_rope_tables_refuses(kw):
    a = dict(max_positions=4, rotary_dim=16, device="cpu")
    a.update(kw)
    with pytest.raises(ValueError):
        nab.rope_tables(**a)


# --------------------------------------------------- join of vocabulary shards --
def _oracle(x, tokens, k, start=0):
    """TokenLogprobs of float64 logits; NaN where a row has no finite entry."""
    lse = x.logsumexp(-1)
    lp = x - lse[:, None]
    at = tokens - start
    inside = (at >= 0) & (at < x.shape[1])
    picked = torch.where(inside, lp.gather(1, torch.where(inside, at, 0)[:, None])[:, 0], -math.inf)
    entropy = -torch.where(lp == -math.inf, 0, lp.exp() * lp).sum(-1)
    order = x.argsort(dim=-1, descending=True, stable=True)[:, :k]
    return nab.TokenLogprobs(picked, entropy, lse, lp.gather(1, order), order + start, x.gather(1, order))


@pytest.mark.parametrize("shards", [1, 2, 5])
def test_join_of_shards_is_the_whole_vocabulary(shards):
    g = torch.Generator().manual_seed(7)
    x = (torch.randn(6, 40 * shards, generator=g, dtype=torch.float64) * 3)
    x = (x * 4).round() / 4  # equal values in different shards
    x[1, 3:] = -math.inf     # all but the first shard masked
    if shards > 1:
        x[2, :40] = -math.inf
    tokens = torch.tensor([0, 1, 40 * shards - 1, 17, 40 * shards // 2, 39])
    whole = _oracle(x, tokens, 7)
    parts = [_oracle(x[:, 40 * i:40 * (i + 1)], tokens, 7, 40 * i) for i in range(shards)]
    got = nab.join_token_logprobs(parts)
    # float64 throughout: a few roundings of values up to 20
    for a, b in zip(got, whole):
        torch.testing.assert_close(a, b, rtol=0, atol=1e-13)


def test_join_of_no_shards():
    with pytest.raises(ValueError):
        nab.join_token_logprobs([])


def _gather(rank, world, port, path):
    import torch.distributed as dist

    dist.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{port}", rank=rank, world_size=world)
    g = torch.Generator().manual_seed(3)
    x = ((torch.randn(4, 50 * world, generator=g, dtype=torch.float64) * 3) * 4).round() / 4
    tokens = torch.tensor([0, 49, 50, 99])
    parts = [_oracle(x[:, 50 * i:50 * (i + 1)], tokens, 5, 50 * i) for i in range(world)]
    got = nab.gather_token_logprobs(parts[rank])
    torch.save((got, nab.join_token_logprobs(parts)), f"{path}/{rank}.pt")
    dist.barrier()
    dist.destroy_process_group()


def test_gather_over_ranks(tmp_path):
    import torch.multiprocessing as mp

    from conftest import free_port

    mp.spawn(_gather, args=(2, free_port(), str(tmp_path)), nprocs=2)
    for rank in range(2):
        got, want = torch.load(tmp_path / f"{rank}.pt", weights_only=False)
        assert torch.equal(got.top_tokens, want.top_tokens)
        for a, b in zip(got, want):
            torch.testing.assert_close(a, b, rtol=0, atol=1e-13)


@pytest.mark.parametrize("kw,match", [
    (dict(kv="pages"), "kv must be"),
    (dict(lengths=[3]), "needs kv='paged'"),
    (dict(kv="paged", page_size=24), "page_size"),
    (dict(kv="paged", page_size=0), "page_size"),
    (dict(kv="paged", max_new=0), "max_new"),
    (dict(kv="paged", lengths=[3, 4]), "one length per request"),
    (dict(kv="paged", lengths=[-1]), "one length per request"),
])
def test_decoder_refuses(kw, match):
    from numa_allreduce_b200.models.llama_tp import LlamaConfig, LlamaTPDecoder

    with pytest.raises(ValueError, match=match):
        LlamaTPDecoder(LlamaConfig.tiny(), None, batch=1, context=4, device="cpu", **kw)


@pytest.mark.parametrize("call, match", [
    (lambda n, t: n.token_logprobs(None, t, 1, 0), "token_logprobs: logits must be a tensor, got NoneType"),
    (lambda n, t: n.token_logprobs(t, [1], 1, 0), "token_logprobs: tokens must be a tensor, got list"),
    (lambda n, t: n.token_logprobs(t, t, 1.5, 0), "token_logprobs: top_k must be a 64-bit integer, got float"),
    (lambda n, t: n.token_logprobs(t, t, 1 << 70, 0), "token_logprobs: top_k must be a 64-bit integer, got int"),
    (lambda n, t: n.token_logprobs(t, t, 1), "token_logprobs takes 4 arguments, got 3"),
    (lambda n, t: n.token_logprobs(), "token_logprobs takes 4 arguments, got 0"),
    (lambda n, t: n.paged_attention(t, t, t, t, t, "1", None), "paged_attention: scale must be a number, got str"),
    (lambda n, t: n.paged_attention(t, t, t, t, t, 1, 2), "paged_attention: out must be a tensor, got int"),
    (lambda n, t: n.assign_pages(t, 3, t, t, t, 16, 1), "assign_pages: query_start must be a tensor, got int"),
    (lambda n, t: n.assign_pages(t, None, t, t, t, 16, None), "assign_pages: num_tokens must be a 64-bit integer"),
    (lambda n, t: n.rope_append_paged(t, t, t, t, t, t, "v", 1, None, None, 0.0, False, None),
     "rope_append_paged: v_pages must be a tensor, got str"),
])
def test_arguments_of_the_wrong_kind(call, match):
    with pytest.raises(TypeError, match=match):
        call(_ext.native(), torch.zeros(1))
