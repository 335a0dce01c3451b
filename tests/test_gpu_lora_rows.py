"""Adapters of more rows than have workgroups of their own for each adapter of a tile (mk_lora_rows, mk_lora_units), and the same results on both sides of that
number."""
import numpy as np
import pytest

from test_gpu_lora import Case

pytestmark = pytest.mark.gpu
MANY = 1025  # (up to 1024 rows tiles of 16)


@pytest.mark.parametrize("xform", ["units", "fp32", "fp16", "bf16"])
@pytest.mark.parametrize("wname", ["fp16", "bf16"])
@pytest.mark.parametrize("rows,n,k,rank,na", [(MANY, 70, 192, 24, 3), (MANY + 6, 33, 64, 7, 40), (1100, 130, 128, 33, 9), (1057, 50, 64, 65, 5), (1280, 200, 64, 16, 1)])
def test_shapes(qkv, torch_gpu, xform, wname, rows, n, k, rank, na):
    Case(torch_gpu, rows, n, k, rank, na, xform, wname, ranks=True, seed=rows + rank, pad=0 if xform == "units" else rows % 4).check(qkv)


@pytest.mark.parametrize("rows", [1000, 1024, MANY, 1060])
def test_ids(qkv, torch_gpu, rows):
    """Every row an adapter of its own, runs, the same everywhere, none anywhere, ids far outside."""
    for ids in (np.arange(rows), np.zeros(rows), np.full(rows, -1), np.full(rows, 2 ** 31 - 1), np.arange(rows) // 130 - 1, (np.arange(rows) * 5) % 6 - 1):
        Case(torch_gpu, rows, 50, 96, 12, rows, ids=ids.astype(np.int64)).check(qkv)


@pytest.mark.parametrize("wname", ["fp16", "bf16"])
@pytest.mark.parametrize("rank", [64, 100, 256])
def test_long_ranks(qkv, torch_gpu, wname, rank):
    Case(torch_gpu, 1100, 70, 64, rank, 4, "bf16", wname, ranks=True, ids=np.arange(1100) // 270 - 1, seed=rank).check(qkv)


def test_parts_of_k(qkv, torch_gpu):
    """Many rows and k in parts, prompts of ragged lengths."""
    Case(torch_gpu, 1500, 300, 2048, 32, 6, "fp32", "bf16", ids=np.sort(np.random.default_rng(2).integers(-1, 6, 1500)), seed=3).check(qkv)
    # (and of rows whose tiles count as four adapters each, one or all of them there)
    Case(torch_gpu, 600, 100, 2048, 20, 6, "bf16", "fp16", ids=np.arange(600) // 200, seed=4).check(qkv)
    Case(torch_gpu, 300, 100, 5120, 20, 80, "units", "bf16", ids=np.arange(300) % 80, seed=5).check(qkv)


def test_in_place_and_base_bits(qkv, torch_gpu):
    """y in place of base; rows without an adapter, and of one of rank 0, are base to the bit."""
    torch, rows = torch_gpu, 1200
    c = Case(torch, rows, 75, 256, 16, 3, "units", ids=np.arange(rows) % 5 - 1, seed=1)
    c.ranks = np.array([16, 0, 9], np.int32)
    c.dev[0] = torch.from_numpy(c.ranks).cuda()
    at = torch.full((rows, 80), 5.0, device="cuda")[:, :75]
    at.copy_(c.dev[3])
    y = c.run(qkv, y=at, base=at)
    ref, bound = c.want()
    assert (np.abs(y.cpu().numpy() - ref) <= bound).all()
    same = [m for m in range(rows) if m % 5 - 1 in (-1, 1, 3)]
    assert torch.equal(y[same], c.dev[3][same])
    assert torch.equal(c.run(qkv), at)  # (out of place: the same bits)


@pytest.mark.parametrize("wname", ["fp16", "bf16"])
def test_not_finite(qkv, torch_gpu, wname):
    """A row's infinities and NaNs stay in it, an adapter's in its rows, and what lies behind its ranks is not used."""
    torch, rows = torch_gpu, 1100
    make = lambda: Case(torch, rows, 70, 128, 20, 3, "fp32", wname, ranks=True, ids=np.arange(rows) % 4 - 1, seed=3)
    c = make()
    c.ranks[:] = [20, 11, 20]
    c.dev[0] = torch.from_numpy(c.ranks).cuda()
    c.a[1, 11:], c.b[1, :, 11:] = float("nan"), float("inf")
    c.check(qkv)
    clean = c.run(qkv).clone()
    c.x[5, 3], c.x[1098, 100] = float("inf"), float("nan")
    y = c.run(qkv)
    rest = [m for m in range(rows) if m not in (5, 1098)]
    assert torch.equal(y[rest], clean[rest]) and not torch.isfinite(y[[5, 1098]]).any()
    c.x[5, 3], c.x[1098, 100] = 1, 1
    clean = c.run(qkv).clone()
    c.a[2, 4, 7] = float("nan")
    y = c.run(qkv)
    hit = [m for m in range(rows) if m % 4 == 3]
    rest = [m for m in range(rows) if m % 4 != 3]
    assert torch.isnan(y[hit]).all() and torch.equal(y[rest], clean[rest])


def test_same_bits_graph(qkv, torch_gpu):
    torch = torch_gpu
    c = Case(torch, 1100, 300, 512, 16, 6, "bf16", seed=5)
    want = c.run(qkv).clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.run(qkv, torch.cuda.current_stream().cuda_stream, ws=c.ws)
    for i in range(4):
        c.y.zero_()
        g.replay()
        torch.cuda.synchronize()
        got = c.y[1:1101, 1:301].clone()
        assert torch.equal(c.run(qkv, ws=c.ws), got) and (i or torch.equal(got, want))
        c.x.mul_(0.5)
        torch.cuda.synchronize()
