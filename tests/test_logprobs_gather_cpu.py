"""The gather of vocabulary shards over gloo ranks carries every token id as it is."""

import pytest
import torch
import torch.distributed as dist

import numa_allreduce_b200 as nab

# ids that no 32-bit float holds, and whose halves are NaN, denormal and negative zero as floats
STARTS = [0, 2 ** 24 + 1, 2 ** 31 - 1, 0x7F800001, 0x1FFC00001, 0x7FF0000000000001 - 2 ** 62, 2 ** 62 + 0x80000000]


def shards(start, k, dtype, world, rows=5):
    g = torch.Generator().manual_seed(k)
    out = []
    for i in range(world):
        x = (torch.randn(rows, 40, generator=g, dtype=torch.float64) * 12).round() / 4
        lse = x.logsumexp(-1)
        values, at = x.sort(dim=-1, descending=True, stable=True)
        lp = values[:, :k] - lse[:, None]
        out.append(nab.TokenLogprobs(x[:, 3].to(dtype), lse.to(dtype) / 9, lse.to(dtype), lp.to(dtype),
                                     at[:, :k] + start + 40 * i, values[:, :k].to(dtype)))
    return out


def _rank(rank, world, port, path):
    dist.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{port}", rank=rank, world_size=world)
    got = [nab.gather_token_logprobs(shards(s, k, dtype, world, rows)[rank])
           for s in STARTS for k in (0, 1, 5) for dtype in (torch.float32, torch.float64) for rows in (0, 1, 5)]
    torch.save(got, f"{path}/{rank}.pt")
    dist.barrier()
    dist.destroy_process_group()


@pytest.mark.parametrize("world", [2])
def test_ids_of_any_size(world, tmp_path):
    import torch.multiprocessing as mp

    from conftest import free_port

    mp.spawn(_rank, args=(world, free_port(), str(tmp_path)), nprocs=world)
    for rank in range(world):
        got = iter(torch.load(tmp_path / f"{rank}.pt", weights_only=False))
        for s in STARTS:
            for k in (0, 1, 5):
                for dtype in (torch.float32, torch.float64):
                    for rows in (0, 1, 5):
                        for a, b in zip(next(got), nab.join_token_logprobs(shards(s, k, dtype, world, rows))):
                            assert a.dtype == b.dtype and torch.equal(a, b)
