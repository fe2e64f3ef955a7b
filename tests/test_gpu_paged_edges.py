"""Paged-cache operators on the GPU at the edges of their ranges: counts,
variants and orders of calls that the sizes of an ordinary batch do not reach.
Oracles and tolerances are those of test_gpu_paged.py."""

import math
import os
import subprocess
import sys

import pytest
import torch

import numa_allreduce_b200 as nab
from test_gpu_paged import BF, FP, attention_oracle, check_attention, gen, make_cache
from test_gpu_paged import clean_record  # noqa: F401 (for every test)

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------- assign_pages --
def test_assign_pages_of_any_count_in_a_new_process():
    """Counts around the shared memory that needs no opting in, where no larger call has opted in before."""
    script = """
import sys, torch
import numa_allreduce_b200 as nab
i32 = dict(dtype=torch.int32, device="cuda")
for b in [int(x) for x in sys.argv[1:]]:
    starts = torch.arange(b + 1, **i32)
    r = nab.assign_pages(torch.full((b,), 16, **i32), torch.zeros(b, 2, **i32), torch.arange(b, **i32),
                         torch.zeros(1, **i32), 16, query_start=starts, num_tokens=b)
    assert r.slots.tolist() == [16 * i for i in range(b)] and r.lengths.eq(17).all(), b
    r = nab.assign_pages(torch.full((b,), 16, **i32), torch.zeros(b, 2, **i32), torch.arange(b, **i32),
                         torch.zeros(1, **i32), 16)
    assert r.slots.tolist() == [16 * i for i in range(b)], b
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    for counts in (["6135", "6136"], ["6140"], ["6143", "6144", "6145"], ["8192"]):
        p = subprocess.run([sys.executable, "-c", script, *counts], cwd=root, capture_output=True, text=True, timeout=300)
        assert p.returncode == 0, p.stderr[-2000:]


# ---------------------------------------------------------- paged_attention --
@pytest.mark.parametrize("batch,cached,page", [(2, 900, 16), (100, 1500, 16), (300, 100, 32)])  # cluster, even, whole
def test_attention_directly_after_assign_pages(batch, cached, page):
    """The table's entries that the launch before has just written, with ids of other pages in their place before."""
    hq, hkv, d = 8, 1, 128
    held, new = -(-cached // page), 2 * page
    width = held + 3
    pages = batch * width
    k = torch.randn(pages, hkv, page, d, generator=gen(1), device="cuda").to(BF)
    v = torch.randn(pages, hkv, page, d, generator=gen(2), device="cuda").to(BF)
    q = torch.randn(batch, hq, d, generator=gen(3), device="cuda").to(BF)
    order = torch.randperm(pages, generator=gen(4), device="cuda").int()
    tables = torch.empty(batch, width, dtype=torch.int32, device="cuda")
    free = order[batch * held:].contiguous()
    n = torch.full((batch,), cached, dtype=torch.int32, device="cuda")
    taken = torch.zeros(1, dtype=torch.int32, device="cuda")
    starts = torch.arange(batch + 1, dtype=torch.int32, device="cuda") * new

    def steps():
        outs = []
        for i in range(6):
            tables.copy_(stale[i])
            step = nab.assign_pages(n, tables, free, taken, page, query_start=starts, num_tokens=batch * new)
            outs.append(nab.paged_attention(q, k, v, tables, step.lengths))
        return outs, step.lengths

    first = order[:batch * held].view(batch, held)
    stale = [torch.cat([first, torch.randint(pages, (batch, 3), generator=gen(5 + i), device="cuda").int()], 1)
             for i in range(6)]
    steps()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs, lengths = steps()
    for _ in range(20):
        graph.replay()
    torch.cuda.synchronize()
    assert lengths.tolist() == [cached + new] * batch
    used = -(-(cached + new) // page) - held
    assert torch.equal(tables[:, held:held + used], free[:batch * used].view(batch, used))
    for out in outs:
        check_attention(out, q, k, v, tables, [cached + new] * batch, d ** -0.5)
    nab.check_kernels()
    del graph


def repeated(lengths, hq, hkv, d, page, dtype, width, seed):
    """Checked against the oracle, and the same bits ten times over."""
    k, v, tables = make_cache(lengths, hkv, d, page, dtype, seed=seed, width=width)
    q = torch.randn(len(lengths), hq, d, generator=gen(seed), device="cuda").to(dtype)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out = nab.paged_attention(q, k, v, tables, n)
    check_attention(out, q, k, v, tables, lengths, 1 / math.sqrt(d))
    for _ in range(10):
        assert torch.equal(nab.paged_attention(q, k, v, tables, n), out)
    nab.check_kernels()


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("lengths,hq,hkv,d,page,width", [
    # even form, few segments cut over many CTAs: one head tile of 9, 12 or 16, two of 9 and 8, three of 14, 13 and 13
    ([2050], 9, 1, 128, 16, None),
    ([3100, 1, 900], 12, 1, 128, 16, None),
    ([8100, 300], 16, 1, 64, 128, None),
    ([6300, 0, 65], 17, 1, 64, 16, None),
    ([9000, 20, 4000, 0, 8999], 32, 2, 128, 48, None),
    # even form, more segments than CTAs
    ([700 + 9 * i for i in range(60)], 40, 2, 128, 64, None),
    ([(97 * i) % 401 for i in range(160)], 24, 2, 128, 16, None),
    ([(97 * i) % 401 for i in range(160)], 8, 2, 128, 16, None),
    # even form, a table far wider than any request: idle CTAs, requests within one CTA
    ([130, 0, 5, 64], 12, 1, 128, 16, 8192),
    ([3000, 0, 5], 8, 2, 64, 64, 2048),
    ([(31 * i) % 500 for i in range(90)], 32, 2, 128, 32, 4096),
    ([1], 8, 1, 128, 16, 1000),
    ([0, 0], 8, 1, 128, 16, 1000),
    # whole segments
    ([(37 * i) % 65 for i in range(300)], 32, 2, 128, 16, None),
    ([(53 * i) % 193 for i in range(200)], 24, 1, 64, 16, None),
    ([(29 * i) % 48 for i in range(400)], 20, 1, 128, 16, None),
    # up to 8 heads in the even and whole forms
    ([5000, 3, 0, 2999], 8, 2, 128, 64, None),
    ([(41 * i) % 129 for i in range(300)], 8, 1, 128, 128, None),
])
def test_every_form_with_few_and_many_heads(lengths, hq, hkv, d, page, width, dtype):
    repeated(lengths, hq, hkv, d, page, dtype, width, seed=len(lengths) + hq)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("batch,n,d,group", [(1, 131071, 64, 8), (40, 16383, 128, 4), (40, 16383, 64, 12)])
@pytest.mark.parametrize("bits", [14, 20, 26, 28])
def test_many_small_probabilities(batch, n, d, group, bits, dtype):
    """Eight early positions outweigh each of the others by 2^bits and add nothing to the output: the others are all
    of it. (Eight, 16 apart: one for every warp. 40 requests of 8 kv heads, with the same pages: each in few CTAs.)"""
    page, hkv, top = 64, 8, 8
    k, v, tables = make_cache([n], hkv, d, page, dtype, seed=bits)
    k[:], v[:] = 0, 1024  # (rows past the length too)
    for i in range(top):
        at = tables[0, 16 * i // page].item()
        k[at, :, 16 * i % page + 3], v[at, :, 16 * i % page + 3] = 1, 0  # scores: d there, 0 elsewhere, exact
    q = torch.ones(batch, hkv * group, d, device="cuda", dtype=dtype)
    scale = bits * math.log(2) / d
    lengths = torch.full((batch,), n, dtype=torch.int32, device="cuda")
    out = nab.paged_attention(q, k, v, tables.expand(batch, -1), lengths, scale=scale)
    want = 1024 * (n - top) / (n - top + top * math.exp(d * torch.tensor(scale, dtype=torch.float32).item()))
    # the probabilities' and the output's rounding; scores, exponentials and sums as in check_attention with exact scores
    # (an exponent of up to 28 with four roundings of 2^-24, an exp2 of 2^-22, for the weight and for the sum)
    u = torch.finfo(dtype).eps / 2
    tol = want * (2 * u + 2 * (28 * 4 * 2 ** -24 + 2 ** -22) + (n / 64 + 64) * 2 ** -22) + torch.finfo(dtype).tiny
    assert (out.double() - want).abs().max().item() <= tol


def exact_scores(lengths, hq, hkv, d, page, dtype, seed):
    """A cache and queries whose scores are sums of whole numbers: exact whatever the order."""
    k, v, tables = make_cache(lengths, hkv, d, page, dtype, seed=seed)
    k.copy_(torch.where(k.isnan(), k, (k * 1.5).round().clamp(-2, 2)))
    q = torch.randint(-2, 3, (len(lengths), hq, d), generator=gen(seed), device="cuda").to(dtype)
    return q, k, v, tables


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("lengths,hq,hkv,d,page", [
    ([3, 5, 17, 64, 200], 8, 2, 128, 16),          # clusters
    ([3, 5, 17, 64, 200], 12, 1, 128, 16),
    ([3, 40, 17, 64, 300], 16, 2, 64, 32),
    ([2100, 3, 900], 4, 1, 128, 16),               # even
    ([2100, 3, 900], 16, 1, 128, 16),
    ([4100, 50, 900], 40, 2, 64, 128),
    ([(37 * i) % 65 for i in range(300)], 8, 1, 128, 16),  # whole
    ([(37 * i) % 65 for i in range(300)], 9, 1, 128, 16),
])
def test_no_rounding_but_the_outputs(lengths, hq, hkv, d, page, dtype):
    """Within the rounding of the output and fp32 work, where the terms cancel too.

    Scores are exact. Their product with scale * log2(e), itself rounded twice, and the difference to the maximum are
    off by 4 V 2^-24 for exponents up to V, exp2 by 2^-22: a weight by 4 V 2^-24 + 2^-22 (ln 2 < 1), and the sum of
    them as much. A probability is held in two 16-bit values, off by u^2; the sums over n positions are as in
    check_attention.
    """
    scale = 0.02
    q, k, v, tables = exact_scores(lengths, hq, hkv, d, page, dtype, seed=len(lengths) + hq)
    out = nab.paged_attention(q, k, v, tables, torch.tensor(lengths, dtype=torch.int32, device="cuda"), scale=scale)
    scale = torch.tensor(scale, dtype=torch.float32).item()
    want, A, qk = attention_oracle(q, k, v, tables, lengths, scale)
    n = torch.tensor(lengths, device="cuda", dtype=torch.float64)[:, None, None]
    u, V = torch.finfo(dtype).eps / 2, 1.4427 * scale * 2 * qk
    own = 2 * (4 * V * 2 ** -24 + 2 ** -22) + u * u + (n / 64 + 64) * 2 ** -22
    tol = u * want.abs() + own * A + torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    err = (out.double() - want).abs()
    assert (err <= tol).all(), f"worst {(err / tol).max().item()} of the tolerance"


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("length,hq", [(100, 8), (100, 12), (5000, 4), (5000, 16)])
def test_infinite_values_stay_infinite(length, hq, dtype):
    """An infinity of v is the output's in its dim; the other dims are as ever."""
    q, k, v, tables = exact_scores([length], hq, 1, 128, 16, dtype, seed=3)
    v[tables[0, 2].item(), 0, 7, 5] = math.inf
    v[tables[0, 4].item(), 0, 1, 9] = -math.inf
    out = nab.paged_attention(q, k, v, tables, torch.tensor([length], dtype=torch.int32, device="cuda"), scale=0.02)
    assert (out[..., 5] == math.inf).all() and (out[..., 9] == -math.inf).all()
    finite = [i for i in range(128) if i not in (5, 9)]
    v[tables[0, 2].item(), 0, 7, 5] = v[tables[0, 4].item(), 0, 1, 9] = 0
    want = nab.paged_attention(q, k, v, tables, torch.tensor([length], dtype=torch.int32, device="cuda"), scale=0.02)
    assert torch.equal(out[..., finite], want[..., finite])


@pytest.mark.parametrize("hq,hkv,dtype,batch,most,form", [
    (8, 2, BF, 7, 6000, "even"), (24, 2, FP, 7, 6000, "even"),      # few segments: descriptors by segment
    (8, 2, BF, 160, 400, "even"), (24, 2, BF, 160, 400, "even"),    # more segments than CTAs
    (32, 2, BF, 300, 64, "whole"), (8, 1, BF, 20, 1000, "cluster"), (24, 1, BF, 20, 1000, "cluster"),
])
def test_a_captured_call_replays_at_any_lengths(hq, hkv, dtype, batch, most, form):
    """Ranges, parts and descriptors are made from the lengths that each replay finds."""
    page, d = 16, 128
    k, v, tables = make_cache([most] * 3, hkv, d, page, dtype, seed=batch)
    k[k.isnan()] = 0  # every row may count: there is one length or another that reaches it
    v[~torch.isfinite(v)] = 0
    tables = tables[torch.arange(batch, device="cuda") % 3].contiguous()
    q = torch.randn(batch, hq, d, generator=gen(batch), device="cuda").to(dtype)
    n = torch.full((batch,), most, dtype=torch.int32, device="cuda")
    nab.paged_attention(q, k, v, tables, n)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = nab.paged_attention(q, k, v, tables, n)
    g = torch.Generator().manual_seed(batch)
    some = torch.randint(0, most + 1, (batch,), generator=g)
    cases = [torch.full((batch,), most), some, torch.zeros(batch, dtype=torch.long), torch.ones(batch, dtype=torch.long),
             torch.where(torch.arange(batch) == batch // 2, most, 0), torch.where(some % 3 == 0, 0, some % 70),
             torch.where(torch.arange(batch) % 2 == 0, most, 1)]
    for lengths in cases:
        n.copy_(lengths)
        graph.replay()
        check_attention(out, q, k, v, tables, lengths.tolist(), d ** -0.5)
        assert torch.equal(out, nab.paged_attention(q, k, v, tables, n))
    nab.check_kernels()
    del graph
