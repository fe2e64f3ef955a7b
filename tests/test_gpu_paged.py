"""Paged-cache decode operators on the GPU against plain float64 (or whole
number) implementations.

Tolerances. u = finfo(type).eps / 2 is the error of one rounding to the
16-bit type, relative to the value; fp32 work adds multiples of 2^-24.
* append: one rounding (u |y|); the fp32 chain before it (sum of squares,
  rsqrt, two products, one sum) stays under 2^-19 of |a| + |b|, the rotated
  pair's magnitudes.
* attention: the output's rounding, u |o|; the probabilities' rounding, u A
  with A = sum_j w_j |v_j|; a score is off by at most d = D 2^-22 scale
  max_j sum |q||k_j| (tensor-core sums may truncate), which moves a weight by
  a factor 1 +- 2 d; the sums over n positions add (n / 64 + 64) 2^-22 A.
"""

import concurrent.futures
import math

import pytest
import torch

import numa_allreduce_b200 as nab

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def clean_record():
    """Every test starts with and (unless it expects one) leaves a clean error record."""
    nab.reset_kernels()
    yield
    nab.reset_kernels()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


# ------------------------------------------------------------- assign_pages --
def assign_oracle(cached, new, tables, free, taken, page, rows):
    """The same with Python loops; `new` None: one token each."""
    width = len(tables[0])
    tables = [list(r) for r in tables]
    positions, slots, lengths = [0] * rows, [-1] * rows, []
    t = 0
    at = min(max(taken, 0), len(free))
    for b, c in enumerate(cached):
        n = 1 if new is None else new[b]
        held = min(-(-c // page), width)
        want = min(-(-(c + n) // page), width)
        have = held
        for j in range(held, want):
            if at < len(free):
                tables[b][j] = free[at]
                at += 1
                have += 1
            else:
                tables[b][j] = -1
        lengths.append(min(c + n, have * page))
        for i in range(n):
            if t < rows:
                p = c + i
                positions[t] = p
                if p // page < want and tables[b][p // page] >= 0:
                    slots[t] = tables[b][p // page] * page + p % page
            t += 1
    return positions, slots, lengths, at, tables


def run_assign(cached, new, page, width, n_free, taken, pad, seed, row_gap=0):
    held = [min(-(-c // page), width) for c in cached]
    total = sum(held) + n_free
    perm = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
    tables, k = [], 0
    for h in held:
        tables.append(perm[k:k + h] + [-7] * (width - h))  # -7: an entry that is not in use
        k += h
    free = perm[k:]
    big = torch.full((len(cached), width + row_gap), -9, dtype=torch.int32, device="cuda")
    dev_tables = big[:, :width]
    dev_tables.copy_(torch.tensor(tables, dtype=torch.int32).reshape(len(cached), width))
    starts = None
    rows = len(cached) + pad
    if new is not None:
        starts = torch.tensor([0] + new).cumsum(0).int().cuda()
        rows = sum(new) + pad
    c = torch.tensor(cached, dtype=torch.int32, device="cuda")
    tk = torch.tensor([taken], dtype=torch.int32, device="cuda")
    for _ in range(2):  # the same call again gives the same: nothing but the tables is changed
        r = nab.assign_pages(c, dev_tables, torch.tensor(free, dtype=torch.int32, device="cuda"), tk, page,
                             query_start=starts, num_tokens=rows if (new is not None or pad) else None)
        want = assign_oracle(cached, new, tables, free, taken, page, rows)
        assert r.positions.tolist() == want[0]
        assert r.slots.tolist() == want[1]
        assert r.lengths.tolist() == want[2]
        assert r.taken.tolist() == [want[3]]
        assert dev_tables.tolist() == want[4]
        assert c.tolist() == cached and tk.tolist() == [taken]
    assert (big[:, width:] == -9).all()


@pytest.mark.parametrize("cached,new,page,width,n_free,taken,pad", [
    ([0], None, 16, 1, 1, 0, 0),
    ([0], [1], 16, 4, 3, 1, 0),
    ([15, 16, 17, 0], None, 16, 3, 8, 2, 5),
    ([5, 64, 0, 33, 7], [0, 40, 0, 1, 0], 32, 6, 9, 0, 3),
    ([3], [1000], 16, 70, 100, 0, 0),
    ([0, 0, 0], [0, 0, 0], 16, 2, 2, 1, 4),
    # the free list ends inside a request, and before one
    ([16, 0, 31], [50, 20, 2], 16, 9, 3, 0, 0),
    ([10, 16], None, 16, 4, 2, 2, 0),
    ([10, 16, 32], None, 16, 4, 2, 99, 0),
    # the table is too narrow
    ([30, 40, 100], [10, 30, 4], 16, 3, 20, 0, 1),
    ([16, 48], [40, 1], 48, 2, 5, 0, 0),
    ([2 ** 31 - 1, 5, 2 ** 31 - 2], None, 16, 3, 4, 0, 1),
])
def test_assign_pages(cached, new, page, width, n_free, taken, pad):
    run_assign(cached, new, page, width, n_free, taken, pad, seed=1)


@pytest.mark.parametrize("batch,cached,new,page,gap", [(33, 500, 1, 16, 0), (513, 70, 3, 16, 5), (1700, 40, 1, 32, 0),
                                                      (97, 900, 300, 128, 3), (8192, 3, 2, 16, 0)])
def test_assign_pages_many_requests(batch, cached, new, page, gap):
    g = torch.Generator().manual_seed(batch)
    c = torch.randint(0, cached + 1, (batch,), generator=g).tolist()
    n = None if new == 1 else torch.randint(0, new + 1, (batch,), generator=g).tolist()
    width = -(-(cached + new) // page) + 1
    need = sum(-(-(a + (1 if n is None else b)) // page) - -(-a // page)
               for a, b in zip(c, n or [1] * batch))
    run_assign(c, n, page, width, need + 3, 2, 11, seed=2, row_gap=gap)
    run_assign(c, n, page, width, max(1, need // 2), 0, 0, seed=3, row_gap=gap)  # half of them fit


# -------------------------------------------------------- rope_append_paged --
def append_oracle(qkv, cos, sin, positions, hq, hkv, d, rotary, interleaved, q_norm, k_norm, eps):
    """q, k, v heads in float64, and |a| + |b| of each rotated pair's members."""
    x = qkv.double().reshape(qkv.shape[0], hq + 2 * hkv, d)
    out, mag = [], []
    for part, w in ((x[:, :hq], q_norm), (x[:, hq:hq + hkv], k_norm)):
        part = part.clone()
        if w is not None:
            part = part / (part.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w.double()
        c, s = cos[positions.long()].double(), sin[positions.long()].double()
        y, m = part.clone(), part.abs()
        for i in range(rotary // 2):
            ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, i + rotary // 2)
            a, b = part[..., ia], part[..., ib]
            y[..., ia] = a * c[:, None, i] - b * s[:, None, i]
            y[..., ib] = b * c[:, None, i] + a * s[:, None, i]
            m[..., ia] = m[..., ib] = a.abs() + b.abs()
        out.append(y)
        mag.append(m)
    return out[0], out[1], x[:, hq + hkv:], mag[0], mag[1]


def check_append(t, hq, hkv, d, rotary, page, dtype, interleaved, q_norm, k_norm, stride_gap=0, seed=0, scale=1.0,
                 skip=True):
    g = gen(seed)
    width = (hq + 2 * hkv) * d
    qkv = (torch.randn(t, width + stride_gap, generator=g, device="cuda") * scale).to(dtype)[:, :width]
    max_pos = 700
    cos, sin = nab.rope_tables(max_pos, rotary, theta=1e4)
    positions = torch.randint(max_pos, (t,), generator=g, device="cuda").int()
    pages = -(-t // page) + 2
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:t]
    if skip and t > 2:
        slots[1::3] = -1
    k0 = torch.randn(pages, hkv, page, d, generator=g, device="cuda").to(dtype)
    v0 = torch.randn(pages, hkv, page, d, generator=g, device="cuda").to(dtype)
    qw = (1 + 0.3 * torch.randn(d, generator=g, device="cuda")).to(dtype) if q_norm else None
    kw = (1 + 0.3 * torch.randn(d, generator=g, device="cuda")).to(dtype) if k_norm else None
    k1, v1 = k0.clone(), v0.clone()
    q = nab.rope_append_paged(qkv, cos, sin, positions, slots, k1, v1, hq, q_norm=qw, k_norm=kw, eps=1e-5,
                              interleaved=interleaved)
    nab.check_kernels()
    wq, wk, wv, mq, mk = append_oracle(qkv, cos, sin, positions, hq, hkv, d, rotary, interleaved, qw, kw, 1e-5)
    u = half_step(dtype)
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps  # a rounding below the normal range
    assert q.shape == (t, hq, d)
    assert ((q.double() - wq).abs() <= u * wq.abs() + 2 ** -19 * mq + tiny).all()
    stored = slots >= 0
    where = slots[stored]
    kr = k1.transpose(1, 2).reshape(-1, hkv, d)
    vr = v1.transpose(1, 2).reshape(-1, hkv, d)
    assert ((kr[where].double() - wk[stored]).abs() <= u * wk[stored].abs() + 2 ** -19 * mk[stored] + tiny).all()
    assert torch.equal(vr[where].double(), wv[stored])
    other = torch.ones(pages * page, dtype=torch.bool, device="cuda")
    other[where] = False
    assert torch.equal(kr[other], k0.transpose(1, 2).reshape(-1, hkv, d)[other])
    assert torch.equal(vr[other], v0.transpose(1, 2).reshape(-1, hkv, d)[other])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("t,hq,hkv,d,rotary,page,dtype,qn,kn,gap", [
    (1, 8, 1, 128, 128, 64, BF, False, False, 0),
    (1, 1, 1, 64, 16, 16, FP, True, True, 0),
    (7, 6, 2, 64, 64, 16, BF, True, True, 8),
    (33, 32, 8, 128, 64, 48, FP, True, False, 0),
    (61, 5, 5, 128, 32, 32, BF, False, True, 40),
    (333, 16, 4, 64, 48, 128, BF, True, True, 0),
    (1025, 3, 1, 128, 112, 16, FP, False, False, 64),
])
def test_rope_append_paged(t, hq, hkv, d, rotary, page, dtype, qn, kn, gap, interleaved):
    check_append(t, hq, hkv, d, rotary, page, dtype, interleaved, qn, kn, gap, seed=t)


@pytest.mark.parametrize("scale", [1e-3, 30.0])
def test_rope_append_paged_small_and_large_values(scale):
    check_append(19, 8, 2, 128, 128, 16, BF, False, True, True, seed=3, scale=scale)


def test_rope_append_paged_matches_the_contiguous_kernel():
    """Same rotation and rows as rope_append at one position for all."""
    from numa_allreduce_b200.ops import _ext

    b, hq, hkv, d, page, pos = 3, 8, 2, 128, 64, 37
    qkv = torch.randn(b, (hq + 2 * hkv) * d, generator=gen(4), device="cuda").to(BF)
    cos, sin = nab.rope_tables(64, d, theta=500000.0)
    kc = torch.zeros(b, hkv, page, d, device="cuda", dtype=BF)
    vc = torch.zeros_like(kc)
    q = torch.empty(b, hq, d, device="cuda", dtype=BF)
    _ext.load().rope_append(qkv, cos, sin, torch.tensor([pos], device="cuda", dtype=torch.int32), q, kc, vc, hq, hkv)
    kp, vp = torch.zeros_like(kc), torch.zeros_like(kc)  # page b belongs to request b
    slots = torch.arange(b, device="cuda") * page + pos
    q2 = nab.rope_append_paged(qkv, cos, sin, torch.full((b,), pos, device="cuda", dtype=torch.int32), slots, kp, vp,
                               hq)
    assert torch.equal(q, q2) and torch.equal(kc, kp) and torch.equal(vc, vp)


def test_rope_append_paged_without_tokens():
    k = torch.zeros(2, 1, 16, 64, device="cuda", dtype=BF)
    cos, sin = nab.rope_tables(4, 64)
    e = torch.zeros(0, device="cuda")
    q = nab.rope_append_paged(torch.zeros(0, 4 * 64, device="cuda", dtype=BF), cos, sin, e.int(), e.long(), k,
                              k.clone(), 2)
    assert q.shape == (0, 2, 64)


def test_rope_append_paged_records_what_is_out_of_range():
    k = torch.zeros(2, 1, 16, 64, device="cuda", dtype=BF)
    v = torch.zeros_like(k)
    cos, sin = nab.rope_tables(4, 64)
    qkv = torch.ones(3, 4 * 64, device="cuda", dtype=BF)
    slots = torch.tensor([0, 32, 2 ** 40], device="cuda")  # the cache has 32 slots
    nab.rope_append_paged(qkv, cos, sin, torch.zeros(3, device="cuda", dtype=torch.int32), slots, k, v, 2)
    with pytest.raises(nab.KernelError, match="out of range"):
        nab.check_kernels()
    assert v[0, 0, 0].eq(1).all() and v.sum().item() == 64  # only the first token is stored
    nab.reset_kernels()
    nab.rope_append_paged(qkv, cos, sin, torch.tensor([0, 4, -1], device="cuda", dtype=torch.int32),
                          torch.arange(3, device="cuda"), k, v, 2)
    with pytest.raises(nab.KernelError, match="out of range"):
        nab.check_kernels()


# ----------------------------------------------------------- paged_attention --
def make_cache(lengths, hkv, d, page, dtype, seed, spare=1, width=None):
    """Pages in random order; unused table entries, and rows past a length, hold what must not matter."""
    g = gen(seed)
    held = [-(-n // page) for n in lengths]
    pages = sum(held) + spare
    k = torch.randn(pages, hkv, page, d, generator=g, device="cuda").to(dtype)
    v = torch.randn(pages, hkv, page, d, generator=g, device="cuda").to(dtype)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    width = width or max(max(held), 1)
    tables = torch.full((len(lengths), width), -5, dtype=torch.int32)
    at = 0
    for b, (n, h) in enumerate(zip(lengths, held)):
        ids = order[at:at + h]
        at += h
        tables[b, :h] = torch.tensor(ids, dtype=torch.int32)
        if n % page:
            k[ids[-1], :, n % page:] = float("nan")
            v[ids[-1], :, n % page:] = float("nan") if b % 2 else float("inf")
    for p in order[at:]:
        k[p] = v[p] = float("nan")
    return k, v, tables.cuda()


def attention_oracle(q, k, v, tables, lengths, scale):
    """Float64 output, and A and the largest sum |q||k| of each head for the tolerance."""
    b_, hq, d = q.shape
    hkv, page = k.shape[1], k.shape[2]
    out = torch.zeros(b_, hq, d, dtype=torch.float64, device=q.device)
    A, qk = torch.zeros_like(out), torch.zeros(b_, hq, 1, dtype=torch.float64, device=q.device)
    for b, n in enumerate(lengths):
        if n == 0:
            continue
        ids = tables[b, :-(-n // page)].long()
        kk = k[ids].transpose(0, 1).reshape(hkv, -1, d)[:, :n].double().repeat_interleave(hq // hkv, 0)
        vv = v[ids].transpose(0, 1).reshape(hkv, -1, d)[:, :n].double().repeat_interleave(hq // hkv, 0)
        w = (torch.einsum("hd,hnd->hn", q[b].double(), kk) * scale).softmax(-1)
        out[b] = torch.einsum("hn,hnd->hd", w, vv)
        A[b] = torch.einsum("hn,hnd->hd", w, vv.abs())
        qk[b] = torch.einsum("hd,hnd->hn", q[b].double().abs(), kk.abs()).amax(-1, keepdim=True)
    return out, A, qk


def check_attention(got, q, k, v, tables, lengths, scale):
    want, A, qk = attention_oracle(q, k, v, tables, lengths, scale)
    u, d = half_step(q.dtype), q.shape[-1] * 2 ** -22 * scale * qk
    n = torch.tensor(lengths, device="cuda", dtype=torch.float64)[:, None, None]
    tol = u * want.abs() + (u + 2 * d + (n / 64 + 64) * 2 ** -22) * A + torch.finfo(q.dtype).tiny
    err = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    assert (err <= tol).all(), f"worst {(err / tol).max().item()} of the tolerance"
    for b, n in enumerate(lengths):
        if n == 0:
            assert (got[b] == 0).all()


@pytest.mark.parametrize("lengths,hq,hkv,d,page,dtype", [
    ([1], 1, 1, 64, 16, BF),
    ([1], 8, 1, 128, 64, FP),
    ([15, 16, 17], 8, 2, 128, 16, BF),
    ([63, 64, 65, 1], 4, 4, 64, 16, FP),
    ([0], 8, 1, 128, 16, BF),
    ([0, 0, 5, 0], 16, 8, 128, 48, BF),
    ([127, 128, 129, 0, 130], 9, 1, 128, 32, BF),     # nine heads: both row halves
    ([200, 1, 77], 32, 2, 128, 128, FP),              # 16 heads of a group
    ([200, 300, 77], 17, 1, 64, 16, BF),              # 17: two head tiles of 9 and 8
    ([513, 40], 40, 1, 128, 64, BF),                  # 40: three head tiles
    ([1025], 8, 1, 128, 64, BF),
    ([4096, 3, 1000, 0, 2049], 28, 4, 128, 256, FP),  # groups of 7
    ([20011], 8, 2, 64, 16, FP),
    ([70000, 1], 8, 1, 128, 64, BF),
])
def test_paged_attention(lengths, hq, hkv, d, page, dtype):
    k, v, tables = make_cache(lengths, hkv, d, page, dtype, seed=len(lengths) + lengths[0])
    q = torch.randn(len(lengths), hq, d, generator=gen(1), device="cuda").to(dtype)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    first = None
    for _ in range(3):
        out = nab.paged_attention(q, k, v, tables, n)
        check_attention(out, q, k, v, tables, lengths, 1 / math.sqrt(d))
        assert first is None or torch.equal(out, first)  # the same bits every time
        first = out
    nab.check_kernels()


@pytest.mark.parametrize("batch,most,hq,hkv,page", [
    (161, 40, 8, 1, 16), (700, 90, 8, 8, 32), (64, 3000, 8, 2, 64), (5, 9000, 64, 8, 16),
    (50, 1500, 64, 8, 64), (50, 1500, 16, 8, 48),   # more segments than CTAs, cut ones among them
    (100, 300, 4, 1, 16), (40, 500, 8, 1, 32), (9, 1100, 12, 1, 64),  # clusters of 2, 4 and 8
    (290, 70, 8, 1, 128), (400, 250, 3, 1, 16),
])
def test_paged_attention_ragged_batches(batch, most, hq, hkv, page):
    """More requests than threads, ranges that begin and end inside requests, requests without positions."""
    g = torch.Generator().manual_seed(batch)
    lengths = torch.randint(0, most + 1, (batch,), generator=g).tolist()
    lengths[batch // 2] = 0
    k, v, tables = make_cache(lengths, hkv, 128, page, BF, seed=batch)
    q = torch.randn(batch, hq, 128, generator=gen(2), device="cuda").to(BF)
    out = nab.paged_attention(q, k, v, tables, torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    check_attention(out, q, k, v, tables, lengths, 128 ** -0.5)
    nab.check_kernels()


@pytest.mark.parametrize("hq,hkv", [(8, 1), (12, 1)])
def test_paged_attention_strided_inputs_scale_and_out(hq, hkv):
    lengths, d, page = [300, 65, 0, 129], 128, 32
    k, v, tables = make_cache(lengths, hkv, d, page, BF, seed=5)
    qkv = torch.randn(4, (hq + 2 * hkv) * d, generator=gen(3), device="cuda").to(BF)
    q = qkv[:, :hq * d].view(4, hq, d)  # rows further apart than the heads
    wide = torch.full((4, tables.shape[1] + 3), 10 ** 6, dtype=torch.int32, device="cuda")
    wide[:, 1:-2] = tables
    out = torch.full((4, hq, d), 7.0, device="cuda", dtype=BF)
    r = nab.paged_attention(q, k, v, wide[:, 1:-2], torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                            scale=0.3, out=out)
    assert r is out
    check_attention(out, q, k, v, tables, lengths, 0.3)


def test_paged_attention_peaked_scores():
    """One position dominates each head by far (scores of hundreds): no overflow, no loss."""
    lengths = [777, 64]
    k, v, tables = make_cache(lengths, 2, 128, 16, BF, seed=6)
    q = (torch.randn(2, 8, 128, generator=gen(4), device="cuda") * 40).to(BF)
    out = nab.paged_attention(q, k, v, tables, torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    check_attention(out, q, k, v, tables, lengths, 128 ** -0.5)


def test_paged_attention_nan_stays_in_its_request():
    lengths = [100, 300, 50]
    k, v, tables = make_cache(lengths, 1, 128, 16, BF, seed=7)
    k[tables[1, 3].item(), 0, 5] = float("nan")
    q = torch.randn(3, 8, 128, generator=gen(5), device="cuda").to(BF)
    out = nab.paged_attention(q, k, v, tables, torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    assert out[1].isnan().all() and torch.isfinite(out[[0, 2]]).all()


def test_paged_attention_shared_pages():
    """Requests that share a prefix point at the same pages; rows of the table may even be one row."""
    k, v, tables = make_cache([200], 2, 64, 16, FP, seed=8)
    q = torch.randn(5, 8, 64, generator=gen(6), device="cuda").to(FP)
    lengths = [200, 1, 100, 0, 199]
    shared = tables.expand(5, -1)
    out = nab.paged_attention(q, k, v, shared, torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    check_attention(out, q, k, v, shared, lengths, 0.125)


def test_paged_attention_records_bad_lengths_and_pages():
    k, v, tables = make_cache([64, 64], 1, 128, 16, BF, seed=9)
    q = torch.randn(2, 8, 128, generator=gen(7), device="cuda").to(BF)
    n = torch.tensor([2 ** 31 - 1, -3], dtype=torch.int32, device="cuda")
    out = nab.paged_attention(q, k, v, tables, n)  # cut to the table's 64, and none
    with pytest.raises(nab.KernelError, match="out of range"):
        nab.check_kernels()
    nab.reset_kernels()
    check_attention(out, q, k, v, tables, [64, 0], 128 ** -0.5)
    nab.check_kernels()
    # a page id outside the cache reads as zeros
    for bad in (-1, k.shape[0], 2 ** 31 - 1, -2 ** 31):
        t = tables.clone()
        t[0, 1] = bad
        out = nab.paged_attention(q, k, v, t, torch.tensor([64, 64], dtype=torch.int32, device="cuda"))
        with pytest.raises(nab.KernelError, match="out of range"):
            nab.check_kernels()
        nab.reset_kernels()
        k2, v2 = (torch.cat([x, torch.zeros_like(x[:1])]) for x in (k, v))
        t[0, 1] = k.shape[0]
        check_attention(out, q, k2, v2, t, [64, 64], 128 ** -0.5)


def test_checks_after_every_launch_on_request(monkeypatch):
    monkeypatch.setenv("NAB_CHECK", "1")
    k, v, tables = make_cache([40], 1, 64, 16, BF, seed=9)
    q = torch.zeros(1, 2, 64, device="cuda", dtype=BF)
    n = torch.tensor([40], dtype=torch.int32, device="cuda")
    nab.paged_attention(q, k, v, tables, n)
    tables[0, 1] = 10 ** 6
    with pytest.raises(nab.KernelError, match="out of range"):
        nab.paged_attention(q, k, v, tables, n)


def test_overlapping_tensors_are_refused():
    pool = torch.zeros(3, 1, 16, 64, device="cuda", dtype=BF)
    cos, sin = nab.rope_tables(4, 64)
    i = torch.zeros(1, device="cuda", dtype=torch.int32)
    q = torch.zeros(1, 2, 64, device="cuda", dtype=BF)
    with pytest.raises(RuntimeError, match="overlap|single memory"):
        nab.paged_attention(q, pool[:2], pool[1:], i[None], i)
    with pytest.raises(RuntimeError, match="overlap|single memory"):
        nab.paged_attention(q, pool, pool.clone(), i[None], i, out=q)
    with pytest.raises(RuntimeError, match="overlap|single memory"):
        nab.rope_append_paged(pool.view(-1)[:256].view(1, 256), cos, sin, i, i.long(), pool, pool.clone(), 2)
    with pytest.raises(RuntimeError, match="overlap|single memory"):
        nab.assign_pages(i, i[None], i, i.clone(), 16)


def test_paged_attention_empty_calls():
    k = torch.zeros(2, 1, 16, 64, device="cuda", dtype=BF)
    out = nab.paged_attention(torch.zeros(0, 4, 64, device="cuda", dtype=BF), k, k.clone(),
                              torch.zeros(0, 3, device="cuda", dtype=torch.int32),
                              torch.zeros(0, device="cuda", dtype=torch.int32))
    assert out.shape == (0, 4, 64)
    out = nab.paged_attention(torch.ones(2, 4, 64, device="cuda", dtype=BF), k, k.clone(),
                              torch.zeros(2, 0, device="cuda", dtype=torch.int32),
                              torch.zeros(2, device="cuda", dtype=torch.int32))
    assert (out == 0).all()


def test_cache_beyond_32_bit_offsets():
    """Pages whose elements lie past 2^31 (and bytes past 2^32) are written and read in place."""
    d, page, hkv, hq = 128, 64, 8, 16
    pages = (1 << 31) // (hkv * page * d) + 40
    k = torch.empty(pages, hkv, page, d, device="cuda", dtype=BF)
    v = torch.empty(pages, hkv, page, d, device="cuda", dtype=BF)
    n = 150
    tables = torch.tensor([[pages - 1, 3, pages - 2]], dtype=torch.int32, device="cuda")
    for p in tables[0].tolist():
        k[p] = torch.randn(hkv, page, d, generator=gen(p), device="cuda").to(BF)
        v[p] = torch.randn(hkv, page, d, generator=gen(p + 1), device="cuda").to(BF)
    qkv = torch.randn(1, (hq + 2 * hkv) * d, generator=gen(8), device="cuda").to(BF)
    cos, sin = nab.rope_tables(200, d)
    step = nab.assign_pages(torch.tensor([n - 1], dtype=torch.int32, device="cuda"), tables,
                            torch.zeros(1, dtype=torch.int32, device="cuda"),
                            torch.zeros(1, dtype=torch.int32, device="cuda"), page)
    assert step.slots.tolist() == [(pages - 2) * page + 21]
    q = nab.rope_append_paged(qkv, cos, sin, step.positions, step.slots, k, v, hq)
    assert torch.equal(v[pages - 2, :, 21], qkv.view(hq + 2 * hkv, d)[hq + hkv:])
    out = nab.paged_attention(q, k, v, tables, step.lengths)
    check_attention(out, q, k, v, tables, [n], d ** -0.5)
    nab.check_kernels()


# ------------------------------------------------------------- run together --
def run_steps(steps, hq, hkv, d, page, dtype, capture):
    """A prompt chunk of different lengths, then decode steps, against contiguous float64 caches."""
    b, layers = 5, 2
    prompt = [7, 0, 33, 16, 1]
    g = gen(11)
    pages, width = 40, 8
    tables = torch.full((b, width), -1, dtype=torch.int32, device="cuda")
    free = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).int().cuda()
    state = torch.zeros(b + 1, dtype=torch.int32, device="cuda")  # cached lengths, then pages taken
    cache = [tuple(torch.full((pages, hkv, page, d), float("nan"), device="cuda", dtype=dtype) for _ in range(2))
             for _ in range(layers)]
    cos, sin = nab.rope_tables(200, d)
    width_qkv = (hq + 2 * hkv) * d
    history = [[[[], []] for _ in range(b)] for _ in range(layers)]

    def remember(layer, rows, positions):
        _, k, v, _, _ = append_oracle(rows, cos, sin, positions, hq, hkv, d, d, False, None, None, 0.0)
        return k.to(dtype), v

    new = [n for n in prompt]
    starts = torch.tensor([0] + new).cumsum(0).int().cuda()
    rows = sum(new) + 3  # three rows of padding
    step = nab.assign_pages(state[:b], tables, free, state[b:], page, query_start=starts, num_tokens=rows)
    for i in range(layers):
        x = torch.randn(rows, width_qkv, generator=g, device="cuda").to(dtype)
        nab.rope_append_paged(x, cos, sin, step.positions, step.slots, *cache[i], hq)
        k, v = remember(i, x, step.positions)
        for r in range(b):
            for t in range(starts[r].item(), starts[r + 1].item()):
                history[i][r][0].append(k[t])
                history[i][r][1].append(v[t])
    state[:b] = step.lengths
    state[b:] = step.taken
    assert state[:b].tolist() == prompt

    static = [torch.empty(b, width_qkv, device="cuda", dtype=dtype) for _ in range(layers)]

    def decode():
        s = nab.assign_pages(state[:b], tables, free, state[b:], page)
        outs = []
        for i in range(layers):
            q = nab.rope_append_paged(static[i], cos, sin, s.positions, s.slots, *cache[i], hq)
            outs.append((q, nab.paged_attention(q, *cache[i], tables, s.lengths)))
        state[:b] = s.lengths
        state[b:] = s.taken
        return outs

    graph = None
    if capture:
        saved = state.clone(), tables.clone()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for x in static:
                x.zero_()
            decode()
        torch.cuda.current_stream().wait_stream(s)
        state.copy_(saved[0])
        tables.copy_(saved[1])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = decode()
    for n in range(steps):
        for i in range(layers):
            static[i].copy_(torch.randn(b, width_qkv, generator=g, device="cuda"))
        before = state[:b].clone()
        if capture:
            graph.replay()
        else:
            outs = decode()
        assert state[:b].tolist() == [p + n + 1 for p in prompt]
        for i in range(layers):
            k, v = remember(i, static[i], before)
            for r in range(b):
                history[i][r][0].append(k[r])
                history[i][r][1].append(v[r])
            q, got = outs[i]
            for r in range(b):
                # this request's own cache, contiguous, as one page
                hist_k = torch.stack(history[i][r][0], 1)[None].to(dtype)
                hist_v = torch.stack(history[i][r][1], 1)[None].to(dtype)
                one = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
                # a stored k may differ from the oracle's by the fp32 chain before its rounding:
                # compare on the cache's own rows where they round to the neighbour
                at = tables[r, :-(-(before[r].item() + 1) // page)].long()
                own = cache[i][0][at].transpose(0, 1).reshape(hkv, -1, d)[:, :before[r].item() + 1][None]
                gap = (own.double() - hist_k.double()).abs()
                assert (gap <= 2 * torch.finfo(dtype).eps * hist_k.double().abs() + 2 ** -18).all()
                assert torch.equal(cache[i][1][at].transpose(0, 1).reshape(hkv, -1, d)[:, :before[r].item() + 1],
                                   hist_v[0])
                check_attention(got[r:r + 1], q[r:r + 1], own, hist_v, one, [before[r].item() + 1], d ** -0.5)
    nab.check_kernels()
    del graph


@pytest.mark.parametrize("capture", [False, True])
@pytest.mark.parametrize("hq,hkv,d,page,dtype", [(8, 2, 128, 16, BF), (6, 1, 64, 16, FP)])
def test_steps_of_a_served_batch(hq, hkv, d, page, dtype, capture):
    run_steps(20, hq, hkv, d, page, dtype, capture)


def test_two_graphs_on_two_streams():
    """Two captured calls replayed at once share nothing."""
    outs, graphs, checks = [], [], []
    for i, lengths in enumerate(([3000, 10, 900], [5000])):
        k, v, tables = make_cache(lengths, 2, 128, 16, BF, seed=20 + i)
        q = torch.randn(len(lengths), 8, 128, generator=gen(30 + i), device="cuda").to(BF)
        n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        nab.paged_attention(q, k, v, tables, n)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(nab.paged_attention(q, k, v, tables, n))
        graphs.append(g)
        checks.append((q, k, v, tables, lengths))
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o, c in zip(outs, checks):
        check_attention(o, *c, 128 ** -0.5)
    nab.check_kernels()
    del graphs


def test_another_stream():
    """Calls made on a stream of their own, inputs made there too."""
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        check_append(65, 8, 2, 128, 128, 16, BF, False, True, True, seed=40)
        lengths = [500, 0, 33]
        k, v, tables = make_cache(lengths, 2, 128, 16, BF, seed=41)
        q = torch.randn(3, 8, 128, generator=gen(42), device="cuda").to(BF)
        out = nab.paged_attention(q, k, v, tables, torch.tensor(lengths, dtype=torch.int32, device="cuda"))
        check_attention(out, q, k, v, tables, lengths, 128 ** -0.5)
    torch.cuda.synchronize()


def test_calls_from_several_threads():
    def work(seed):
        lengths = [300 + 7 * seed, 0, 33]
        k, v, tables = make_cache(lengths, 2, 64, 16, BF, seed=seed)
        q = torch.randn(3, 4, 64, generator=torch.Generator().manual_seed(seed)).to("cuda", BF)
        n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        with torch.cuda.stream(torch.cuda.Stream()):
            outs = [nab.paged_attention(q, k, v, tables, n) for _ in range(50)]
            torch.cuda.current_stream().synchronize()
        return outs, q, k, v, tables, lengths

    with concurrent.futures.ThreadPoolExecutor(4) as pool:
        for outs, q, k, v, tables, lengths in pool.map(work, range(4)):
            check_attention(outs[0], q, k, v, tables, lengths, 64 ** -0.5)
            assert all(torch.equal(o, outs[0]) for o in outs[1:])
