"""Workspaces of the adapters, the router and the experts, without a GPU: what the size functions give for a batch serves every smaller one."""
import pytest

from test_host_mix import lora, moe, route

ROWS = [0, 1, 2, 3, 5, 8, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 80, 100, 127, 128, 129, 160, 200, 255, 256, 257, 288, 292, 293, 300, 341, 342, 400, 409, 410, 511, 512, 513, 600, 682, 683,
        900, 1023, 1024, 1025, 1200, 2000, 2048, 2049, 4000, 4095, 4096]
LONG = [5000, 5461, 5462, 8191, 8192, 8193, 16384, 16385, 70000, 1 << 19]


def workspace_refused(call):
    """Whether the call is refused for its workspace (else, without device memory, for its addresses, which are looked at later)."""
    try:
        call()
    except Exception as e:
        return "workspace" in str(e)
    return False


@pytest.mark.parametrize("k,rank", [(32, 16), (64, 1), (2048, 24), (5120, 16), (5120, 256), (17408, 64), (1 << 20, 100)])
def test_lora(qkv, k, rank):
    at = ROWS + LONG
    need = [qkv.lora_ws(r, k, rank) for r in at]
    assert need == sorted(need) and need[0] == 0
    for i, r in enumerate(at[1:], 1):
        for j in (i, i + 1, i + 3, len(at) - 1):  # of as many rows, of a few more, of the most
            size = need[min(j, len(at) - 1)]
            assert not workspace_refused(lambda: lora(qkv, rows=r, k=k, xs=k, rank=rank, size=size))


@pytest.mark.parametrize("dim,e", [(1, 1), (64, 8), (2048, 128), (5120, 16), (5120, 60), (5120, 256), (7168, 257), (1 << 17, 1024)])
def test_route(qkv, dim, e):
    at = ROWS + LONG
    need = [qkv.moe_route_ws(r, dim, e) for r in at]
    assert need == sorted(need) and need[0] == 0
    for i, r in enumerate(at[1:], 1):
        for j in (i, i + 1, i + 3, len(at) - 1):
            size = need[min(j, len(at) - 1)]
            assert not workspace_refused(lambda: route(qkv, rows=r, dim=dim, xs=dim, e=e, top=1, size=size))


@pytest.mark.parametrize("dim,inner,e,top", [(64, 64, 8, 2), (2048, 768, 128, 8), (5120, 1536, 256, 8), (5120, 6144, 8, 2), (4096, 8192, 16, 1), (16384, 32, 300, 4)])
def test_moe(qkv, dim, inner, e, top):
    need = [qkv.moe_ws(r, dim, inner, e, top) for r in ROWS]
    assert need == sorted(need)
    for i, r in enumerate(ROWS[1:], 1):
        for j in (i, i + 1, i + 3, len(ROWS) - 1):
            size = need[min(j, len(ROWS) - 1)]
            for form in ("rows", "units", "layer"):
                assert not workspace_refused(lambda: moe(qkv, form, rows=r, dim=dim, inner=inner, e=e, top=top, xs=dim, ys=dim, size=size))


def test_the_shapes_have_parts(qkv):
    """Shapes above for which a batch's own need falls where it grows: partial sums that larger batches do not have."""
    assert qkv.moe_route_ws(4096, 2048, 128) >= 8 * 128 * 256 * 4 > 0
    assert qkv.lora_ws(33, 17408, 64) >= qkv.lora_ws(32, 17408, 64) >= 32 * 64 * 4 * 2
