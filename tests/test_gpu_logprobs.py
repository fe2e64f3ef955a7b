"""Token log-probabilities on the GPU against float64.

Tolerances: a term exp(x - m) is off by a few 2^-23 times 1 + |log2 of it|
(weighted by the term itself, at most 2 on average), and a sum of V terms in
512 running sums adds V / 512 roundings and a tree of about 40: together
r = (64 + V / 512) 2^-23 of S. lse = m + log S and logprob = x - lse are then
off by r and a few roundings (2^-22) of their own parts; the entropy by
r (1 + log V) in the weighted mean and r in log S, doubled.
"""

import math

import pytest
import torch

import numa_allreduce_b200 as nab

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def check(x, tokens, k, start=0):
    r = nab.token_logprobs(x, tokens, top_k=k, vocab_start=start)
    rows, v = x.shape
    y = x.double()
    m = y.amax(-1, keepdim=True)
    log_s = (y - m).exp().sum(-1, keepdim=True).log()
    lse = (m + log_s)[:, 0]
    lp = (y - m) - log_s  # not y - lse: at the lowest values of a type log_s is lost in m
    entropy = -torch.where(lp == -math.inf, 0, lp.exp() * lp).sum(-1)
    at = tokens - start
    inside = (at >= 0) & (at < v)
    want = torch.where(inside, lp.gather(1, torch.where(inside, at, 0)[:, None])[:, 0], -math.inf)
    values, ids = y.sort(dim=-1, descending=True, stable=True)
    rel = (64 + v / 512) * 2 ** -23
    assert r.logprob.shape == r.entropy.shape == r.lse.shape == (rows,)
    assert r.top_logprobs.shape == r.top_tokens.shape == (rows, k)
    assert torch.equal(r.top_tokens, ids[:, :k] + start)
    assert torch.equal(r.top_logits.double(), values[:, :k])

    def near(got, exact, tol):
        exact = torch.where(exact.abs() > torch.finfo(F32).max, exact.sign() * math.inf, exact)  # fp32 has no such value
        fine = torch.isfinite(exact)
        assert torch.equal(got.double()[~fine], exact[~fine])
        err = (got.double() - exact).abs()[fine]
        assert (err <= tol.expand_as(exact)[fine]).all(), f"worst {(err / tol.expand_as(exact)[fine]).max().item()}"

    own = 2 ** -22 * (lse.abs() + y.amax(-1).abs())
    near(r.lse, lse, rel + own)
    near(r.logprob, want, rel + own + 2 ** -22 * torch.where(torch.isfinite(want), want, 0).abs())
    near(r.entropy, entropy, torch.full_like(entropy, 2 * rel * (2 + math.log(v))))
    top = (values[:, :k] - m) - log_s
    near(r.top_logprobs, top, (rel + own)[:, None] + 2 ** -22 * torch.where(torch.isfinite(top), top, 0).abs())
    return r


def logits(rows, v, dtype, seed, scale=2.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(rows, v, generator=g, device="cuda") * scale).to(dtype)


def tokens(rows, v, seed=1):
    return torch.randint(v, (rows,), generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("rows,v,k", [(1, 128256, 20), (1, 1, 1), (2, 3, 3), (3, 7, 0), (5, 100, 32), (1, 33, 32),
                                      (4, 4095, 5), (33, 16032, 8), (300, 5001, 20), (2, 262145, 32),
                                      (700, 2048, 1), (16, 4096, 32), (17, 8193, 32)])
def test_token_logprobs(rows, v, k, dtype):
    check(logits(rows, v, dtype, rows + v), tokens(rows, v), k)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,v,k", [(149, 30001, 5), (148, 30001, 5), (148, 8191, 32), (75, 47999, 3), (74, 24001, 32),
                                      (37, 50003, 20), (18, 100003, 32), (18, 96001, 1), (9, 200003, 7), (9, 12001, 0)])
def test_rows_shared_by_several_ctas_and_not(rows, v, k, dtype):
    check(logits(rows, v, dtype, rows + v), tokens(rows, v), k)


@pytest.mark.parametrize("copies", [6, 20, 60])
def test_more_large_values_than_are_collected(copies):
    v = 131072
    x = logits(2, v, F32, 8, 1.0)
    i = torch.arange(v, device="cuda")
    hot = (i % 4096) < 64
    x[:, hot] = 50 + (i[hot] * 7919 % 2048).float() / 64
    check(x.repeat(copies, 1), tokens(2 * copies, v), 32)


@pytest.mark.parametrize("dtype,offset", [(BF, 1), (BF, 7), (FP, 3), (F32, 1), (F32, 3)])
def test_rows_of_any_alignment(dtype, offset):
    big = logits(9, 5003 + 20, dtype, 3)
    check(big[:, offset:offset + 5003], tokens(9, 5003), 16)


@pytest.mark.parametrize("start", [0, 16032, 5 * 16032])
def test_a_shard_of_the_vocabulary(start):
    t = tokens(40, 8 * 16032)
    check(logits(40, 16032, BF, 4), t, 8, start=start)


def test_tokens_outside_the_vocabulary():
    t = torch.tensor([-1, -100, 50, 2 ** 62], device="cuda")
    r = check(logits(4, 50, F32, 5), t, 3)
    assert (r.logprob == -math.inf).all()
    far = torch.tensor([-2 ** 63, 2 ** 63 - 1, 6, 7], device="cuda")
    r = nab.token_logprobs(logits(4, 50, F32, 5), far, vocab_start=7)
    assert (r.logprob[:3] == -math.inf).all() and torch.isfinite(r.logprob[3])


@pytest.mark.parametrize("v", [50, 4096, 40000])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_equal_values_rank_by_the_lowest_token(v, dtype):
    x = torch.full((3, v), 1.5, device="cuda", dtype=dtype)
    x[1] = torch.arange(v, device="cuda") % 3
    x[2, v // 2:] = 2.0
    check(x, tokens(3, v), 32)


@pytest.mark.parametrize("order", ["rising", "falling", "comb"])
def test_contrived_orders(order):
    """Sorted rows, and rows whose large values all fall to a few threads (more than the collection holds)."""
    v = 131072
    if order == "comb":
        x = logits(2, v, F32, 6, 1.0)
        x[:, ::4096] = 100 + torch.arange(v // 4096, device="cuda").float()
        # 8 threads' worth of columns hold thousands of large, all different values
        i = torch.arange(v, device="cuda")
        hot = (i % 2048) < 32
        x[:, hot] = 50 + (i[hot] * 7919 % 2048).float() / 64
    else:
        x = torch.arange(v, device="cuda").float()[None].repeat(2, 1) / 4096
        x = x if order == "rising" else x.flip(1).contiguous()
    check(x, tokens(2, v), 32)
    check(x.repeat(300, 1), tokens(600, v), 20)  # one CTA per row


@pytest.mark.parametrize("dtype", [BF, FP, F32])
def test_masked_entries(dtype):
    """-inf and the type's lowest value: probability 0; few or one token left; whole rows at the lowest value."""
    v = 9000
    low = torch.finfo(dtype).min
    x = logits(6, v, dtype, 7)
    x[0, 100:] = -math.inf
    x[1, 3:] = low
    x[2] = -math.inf
    x[2, 4321] = 0.25
    x[3] = low
    x[4, ::2] = -math.inf
    x[5, :] = low
    x[5, 8999] = torch.finfo(dtype).max
    r = check(x, torch.tensor([5, 1, 4321, 17, 1, 8999], device="cuda"), 20)
    assert r.logprob[2].item() == 0 and r.entropy[2].item() == 0
    assert r.top_tokens[2].tolist() == [4321] + list(range(19))


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("mask", [-1e3, -3e4, -1e9, -1e20, -1e30, -3e38])
def test_finite_masks(mask, dtype):
    """All but one or a few tokens, or all of them, at a finite value far below."""
    if dtype == FP and mask < -6e4:
        mask = -6.5e4
    for v in (3000, 40000):
        x = torch.full((4, v), mask, device="cuda", dtype=dtype)
        x[0, v - 5] = 1.0
        x[1, 10:14] = torch.tensor([0.5, 2.0, -3.0, 2.0], device="cuda", dtype=dtype)
        x[2] = -math.inf
        x[2, ::2] = mask
        check(x, torch.tensor([v - 5, 12, 4, 100], device="cuda"), 20)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("scale", [1e3, 1e6, 1e7, 3e7, 1e12, 1e30])
def test_large_logits(scale, dtype):
    check(logits(5, 20000, dtype, 14, scale), tokens(5, 20000), 10)


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("v", [5000, 70000])
def test_rows_near_the_ends_of_the_type(v, dtype):
    """Maxima around the values where the sums change form, with masked entries beside them."""
    top = torch.finfo(dtype).max
    x = logits(10, v, dtype, 13)
    for i, m in enumerate((-0.97, -0.7, -0.45, -0.2, -0.13, -0.1, 0.1, 0.2, 0.4, 0.97)):
        x[i] = torch.finfo(dtype).min if i % 2 else -math.inf
        x[i, 7::3] = top * m
    check(x, tokens(10, v), 20)


@pytest.mark.parametrize("dtype", [BF, FP, F32])
def test_rows_without_a_distribution(dtype):
    x = logits(5, 5000, dtype, 8)
    x[0] = -math.inf
    x[1, 77] = math.nan
    x[2, 78] = math.inf
    x[3] = math.nan
    r = nab.token_logprobs(x, tokens(5, 5000), top_k=4)
    assert r.logprob[:4].isnan().all() and r.entropy[:4].isnan().all()
    assert r.lse[0] == -math.inf and r.lse[1:4].isnan().all()
    assert torch.isfinite(r.logprob[4]) and torch.isfinite(r.top_logprobs[4]).all()
    assert r.top_tokens[0].tolist() == [0, 1, 2, 3] and r.top_tokens[3].tolist() == [0, 1, 2, 3]
    assert r.top_tokens[2, 0].item() == 78
    order = torch.where(x[1].isnan(), -math.inf, x[1]).sort(descending=True, stable=True)[1]
    assert r.top_tokens[1].tolist() == order[:4].tolist()


def test_no_rows():
    r = nab.token_logprobs(torch.zeros(0, 10, device="cuda"), torch.zeros(0, device="cuda", dtype=torch.long), top_k=2)
    assert r.logprob.shape == (0,) and r.top_tokens.shape == (0, 2)


def test_shards_joined_are_the_whole():
    x = logits(20, 8 * 2000, BF, 9)
    t = tokens(20, 8 * 2000)
    whole = check(x, t, 20)
    parts = [nab.token_logprobs(x[:, i * 2000:(i + 1) * 2000], t, top_k=20, vocab_start=i * 2000) for i in range(8)]
    got = nab.join_token_logprobs(parts)
    # both are within the module's tolerance of the exact values; the join adds a few fp32 roundings of values to 20
    tol = 2 * (64 + 16000 / 512) * 2 ** -23 * (2 + math.log(16000)) * 2 + 20 * 2 ** -21
    for a, b in zip(got, whole):
        if a.dtype == torch.long:
            assert torch.equal(a, b)
        else:
            assert ((a - b).abs() <= tol).all()


def test_captured_and_replayed():
    x, t = logits(3, 70000, BF, 10), tokens(3, 70000)
    nab.token_logprobs(x, t, top_k=5)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r = nab.token_logprobs(x, t, top_k=5)
    x.copy_(logits(3, 70000, BF, 11))
    t.copy_(tokens(3, 70000, 12))
    g.replay()
    torch.cuda.synchronize()
    want = nab.token_logprobs(x, t, top_k=5)
    for a, b in zip(r, want):
        assert torch.equal(a, b)  # the same sums in the same order
    check(x, t, 5)
    del g
