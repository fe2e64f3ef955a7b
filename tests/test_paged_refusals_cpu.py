"""Calls of the paged-cache operators and the token log-probabilities that must
be refused before anything is launched: tensors that share memory with one
that the call writes."""

import pytest
import torch

import numa_allreduce_b200 as nab

BF = torch.bfloat16


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def as_type(raw, dtype, offset, *shape):
    """A tensor in the bytes of `raw` from `offset` on."""
    n = torch.Size(shape).numel() * dtype.itemsize
    return raw.view(-1).view(torch.uint8)[offset:offset + n].view(dtype).view(shape)


def append(**kw):
    a = dict(qkv=torch.zeros(3, 8 * 64, dtype=BF), cos=torch.zeros(10, 32), sin=torch.zeros(10, 32),
             positions=i32(3), slots=torch.arange(3), k_pages=torch.zeros(2, 2, 16, 64, dtype=BF),
             v_pages=torch.zeros(2, 2, 16, 64, dtype=BF), q_heads=4)
    a.update(kw)
    return nab.rope_append_paged(**a)


def attend(**kw):
    a = dict(q=torch.zeros(2, 4, 64, dtype=BF), k_pages=torch.zeros(3, 2, 16, 64, dtype=BF),
             v_pages=torch.zeros(3, 2, 16, 64, dtype=BF), block_tables=i32(2, 3), lengths=i32(2))
    a.update(kw)
    return nab.paged_attention(**a)


def assign(**kw):
    a = dict(cached=i32(2), block_tables=i32(2, 4), free_pages=i32(3), taken=i32(1), page_size=16)
    a.update(kw)
    return nab.assign_pages(**a)


def refused(call, match="overlap"):
    with pytest.raises(RuntimeError, match=match):
        call()


# --------------------------------------------------------- shared memory --
def test_append_does_not_write_what_it_reads():
    pool = torch.zeros(1 << 15, dtype=BF)
    pages = pool[:4096].view(2, 2, 16, 64)
    for name in ("k_pages", "v_pages"):
        kw = {name: pages}
        refused(lambda: append(qkv=pool[1024:1024 + 1536].view(3, 512), **kw))
        refused(lambda: append(cos=as_type(pool, torch.float32, 4096, 10, 32), **kw))
        refused(lambda: append(sin=as_type(pool, torch.float32, 0, 10, 32), **kw))
        refused(lambda: append(positions=as_type(pool, torch.int32, 8188, 3), **kw))
        refused(lambda: append(slots=as_type(pool, torch.int64, 64, 3), **kw))
        refused(lambda: append(q_norm=pool[64:128], **kw))
        refused(lambda: append(k_norm=pool[4032:4096], **kw))
        refused(lambda: append(out=pool[3840:3840 + 768].view(3, 4, 64), **kw))
        # right behind the pages: not refused for that
        refused(lambda: append(qkv=pool[4096:4096 + 1536].view(3, 512), out=pool[8192:8192 + 768].view(3, 4, 64), **kw),
                "must be a CUDA tensor")
    refused(lambda: append(k_pages=pages, v_pages=pool[2048:2048 + 4096].view(2, 2, 16, 64)))
    out = pool[8192:8192 + 768].view(3, 4, 64)
    refused(lambda: append(out=out, qkv=pool[8192:8192 + 1536].view(3, 512)))
    refused(lambda: append(out=out, slots=as_type(pool, torch.int64, 2 * 8192, 3)))


def test_append_with_rows_apart():
    """Rows of qkv further apart than their width: what lies between them is free for other tensors."""
    wide = torch.zeros(3, 4096, dtype=BF)
    qkv = wide[:, 1024:1024 + 512]
    flat = wide.view(-1)
    refused(lambda: append(qkv=qkv, out=flat[4096 + 1024 + 504:][:768].view(3, 4, 64)))  # the end of the second row
    refused(lambda: append(qkv=qkv, out=flat[2 * 4096 + 512:][:768].view(3, 4, 64)))     # up to the third row's start
    refused(lambda: append(qkv=qkv, k_pages=flat[:4096].view(2, 2, 16, 64)))
    refused(lambda: append(qkv=qkv, out=flat[2048:][:768].view(3, 4, 64)), "must be a CUDA tensor")
    refused(lambda: append(qkv=qkv, out=flat[4096 + 256:][:768].view(3, 4, 64)), "must be a CUDA tensor")
    refused(lambda: append(qkv=qkv, out=flat[8192 + 1536:][:768].view(3, 4, 64)), "must be a CUDA tensor")


def test_attention_does_not_write_what_it_reads():
    pool = torch.zeros(1 << 14, dtype=BF)
    out = pool[1024:1536].view(2, 4, 64)
    refused(lambda: attend(out=out, q=pool[1024:1536].view(2, 4, 64)))
    wide = torch.zeros(2, 1024, dtype=BF)
    refused(lambda: attend(q=wide[:, :256].view(2, 4, 64), out=wide.view(-1)[768:1280].view(2, 4, 64)))
    refused(lambda: attend(q=wide[:, :256].view(2, 4, 64), out=wide.view(-1)[256:768].view(2, 4, 64)),
            "must be a CUDA tensor")
    refused(lambda: attend(out=out, k_pages=pool[:6144].view(3, 2, 16, 64)))
    refused(lambda: attend(out=out, v_pages=pool[1528:][:6144].view(3, 2, 16, 64)))
    refused(lambda: attend(out=out, block_tables=as_type(pool, torch.int32, 2048, 2, 3)))
    refused(lambda: attend(out=out, lengths=as_type(pool, torch.int32, 3064, 2)))


def test_assign_pages_does_not_write_what_it_reads():
    wide = i32(2, 16)
    flat = wide.view(-1)
    tables = wide[:, 4:8]
    refused(lambda: assign(block_tables=tables, cached=flat[20:22]))
    refused(lambda: assign(block_tables=tables, taken=flat[7:8]))
    refused(lambda: assign(block_tables=tables, free_pages=flat[1:5]))
    refused(lambda: assign(block_tables=tables, query_start=flat[18:21], num_tokens=2))
    # between the rows of the table
    refused(lambda: assign(block_tables=tables, cached=flat[0:2], taken=flat[3:4], free_pages=flat[8:20],
                           query_start=flat[24:27], num_tokens=2), "must be a CUDA tensor")


# ------------------------------------------ tensors that are not plain memory --
def logprobs(**kw):
    a = dict(logits=torch.zeros(2, 10), tokens=torch.zeros(2, dtype=torch.int64), top_k=3)
    a.update(kw)
    return nab.token_logprobs(**a)


def test_forward_mode_tangents_are_refused():
    import torch.autograd.forward_ad as fw

    with fw.dual_level():
        def dual(*shape, dtype=BF):
            return fw.make_dual(torch.zeros(*shape, dtype=dtype), torch.ones(*shape, dtype=dtype))

        refused(lambda: logprobs(logits=dual(2, 10, dtype=torch.float32)), "logits.*tangent")
        refused(lambda: append(qkv=dual(3, 512)), "qkv.*tangent")
        refused(lambda: append(k_norm=dual(64)), "k_norm.*tangent")
        refused(lambda: append(k_pages=dual(2, 2, 16, 64)), "k_pages.*tangent")
        refused(lambda: attend(q=dual(2, 4, 64)), "q .*tangent")
        refused(lambda: attend(v_pages=dual(3, 2, 16, 64)), "v_pages.*tangent")
        refused(lambda: attend(out=dual(2, 4, 64)), "out.*tangent")
        with torch.no_grad():
            refused(lambda: attend(q=dual(2, 4, 64)), "q .*tangent")


def test_tensors_without_memory_of_their_own_are_refused():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        fake = torch.empty(2, 10, device="cuda"), torch.empty(2, 4, 64, dtype=BF, device="cuda")
    refused(lambda: logprobs(logits=fake[0]), "logits must be a plain tensor")
    refused(lambda: attend(q=fake[1]), "q must be a plain tensor")
    refused(lambda: attend(out=fake[1]), "out must be a plain tensor")
    refused(lambda: logprobs(logits=torch.zeros(2, 10, device="meta")), "logits must be a plain tensor")
    refused(lambda: logprobs(logits=torch.zeros(2, 10).to_sparse()), "logits must be a plain tensor")
    refused(lambda: logprobs(logits=torch._neg_view(torch.zeros(2, 10))), "logits must be a plain tensor")
    refused(lambda: logprobs(logits=torch._efficientzerotensor(2, 10)), "logits must be a plain tensor")
    refused(lambda: torch.vmap(lambda x: logprobs(logits=x).logprob)(torch.zeros(4, 2, 10)), "plain tensor")
    refused(lambda: torch.func.jvp(lambda x: logprobs(logits=x).logprob, (torch.zeros(2, 10),), (torch.ones(2, 10),)),
            "plain tensor|tangent")
    refused(lambda: torch.func.functionalize(lambda x: logprobs(logits=x).logprob)(torch.zeros(2, 10)), "plain tensor")

    class Wrapped(torch.Tensor):
        @classmethod
        def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    refused(lambda: logprobs(logits=torch.zeros(2, 10).as_subclass(Wrapped)), "logits must be a plain tensor")
    refused(lambda: logprobs(logits=torch.nn.Parameter(torch.zeros(2, 10), requires_grad=False)),
            "must be a CUDA tensor")  # a parameter is one


# ------------------------------------------------------------------ sizes --
def test_a_table_for_more_positions_than_fit_32_bits():
    """The tiles of a request are counted from its length and a tile in 32 bits (the tensors are never touched)."""
    refused(lambda: attend(block_tables=torch.empty(2, 2 ** 27, dtype=torch.int32)), "too wide")
    refused(lambda: attend(block_tables=torch.empty(2, 2 ** 27 - 1, dtype=torch.int32)), "too wide")
    refused(lambda: attend(block_tables=torch.empty(2, 2 ** 27 - 8, dtype=torch.int32)), "must be a CUDA tensor")


# ------------------------------------------------------ checks on request --
def test_checks_look_at_the_tensors_device(monkeypatch):
    """With NAB_CHECK=1 a call checks the record of the device that it ran on, whichever device is current."""
    from numa_allreduce_b200.ops import errors, logprobs as lp, paged

    seen = []

    class Device:
        def __init__(self, device):
            seen.append(device)

        def __enter__(self):
            seen.append("in")

        def __exit__(self, *a):
            seen.append("out")

    class Native:
        def check_requested(self):
            return True

        def assign_pages(self, *a):
            return a[:4]

        def rope_append_paged(self, *a):
            return a[0]

        def paged_attention(self, *a):
            return a[0]

        def token_logprobs(self, *a):
            return [a[0]] * 6

    class OnAnotherGpu:
        device, shape = torch.device("cuda", 3), (2, 4, 64)

    monkeypatch.setenv("NAB_CHECK", "1")
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(errors, "check_kernels", lambda sync=True: seen.append("checked"))
    for module in (lp, paged):
        monkeypatch.setattr(module._ext, "native", Native)
    t = OnAnotherGpu()
    for call in (lambda: nab.assign_pages(t, t, t, t, 16), lambda: nab.rope_append_paged(t, t, t, t, t, t, t, 1),
                 lambda: nab.paged_attention(t, t, t, t, t), lambda: nab.token_logprobs(t, t)):
        seen.clear()
        call()
        assert seen == [t.device, "in", "checked", "out"]


# ------------------------------------------------- what is not to be refused --
def test_one_row_of_any_stride():
    """The stride of a single row says nothing."""
    refused(lambda: append(qkv=torch.zeros(512, 1, dtype=BF).t(), positions=i32(1), slots=torch.arange(1)),
            "must be a CUDA tensor")
    refused(lambda: append(qkv=torch.zeros(516, dtype=BF).as_strided((1, 512), (4, 1)), positions=i32(1),
                           slots=torch.arange(1)), "must be a CUDA tensor")


def test_the_default_scale_needs_no_shape():
    """A bad q is refused with its name without a scale too."""
    refused(lambda: attend(q=torch.zeros((), dtype=BF)), "paged_attention: q must be")
    refused(lambda: attend(q=torch.zeros(2, 4, 0, dtype=BF)), "paged_attention: q must be")
    with pytest.raises(TypeError, match="paged_attention: q must be a tensor, got NoneType"):
        attend(q=None)
    with pytest.raises(TypeError, match="paged_attention: scale must be a number, got str"):
        attend(scale="1")
