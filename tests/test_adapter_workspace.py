"""The workspace of the adapters' gradients: what it asks for, without a GPU."""
from __future__ import annotations

import pytest

from hmoe import capi

LIMIT = 1 << 30


def _bytes(adapters, rows, left, right):
    return capi.load().hm_adapter_weight_grad_workspace_bytes(adapters, rows, left, right)


@pytest.mark.parametrize("adapters", [1, 4, 32, 300, 1000, 10000, 65535])
def test_stays_small(adapters):
    """Beside many adapters' gradients the parts' sums stay within 1 GB: they were up to 64 times the gradients."""
    for left, right in ((8, 2048), (16, 4096), (4096, 16), (64, 64), (256, 8192), (1, 1)):
        for rows in (1, 257, 4096, 100000, (1 << 23) - 1):
            assert _bytes(adapters, rows, left, right) <= LIMIT, (left, right, rows)


def test_few_adapters_are_cut():
    """Where parts are few and small they are as many as fill the chip."""
    for adapters, rows, left, right, parts in ((4, 2048, 16, 2048, 8), (4, 2048, 2048, 16, 8), (1, 1 << 20, 64, 64, 64),
                                               (32, 4096, 64, 2048, 16)):
        assert _bytes(adapters, rows, left, right) == parts * adapters * (left * right + 1) * 4


@pytest.mark.gpu
@pytest.mark.parametrize("adapters,rows,left,right", [(3000, 2100, 16, 2048), (600, 1500, 1024, 16), (20000, 600, 8, 520)])
def test_many_adapters(dev, adapters, rows, left, right):
    """Gradients of many adapters, fewer parts than the rows would give, against the formula in 64 bits."""
    import grouped_ref as R
    from hmoe import adapters as A
    torch = dev.torch
    g = torch.Generator(device="cuda")
    g.manual_seed(rows)
    l = torch.empty(rows, left, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    r = torch.empty(rows, right, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    # a few adapters of many rows, most of one or none
    ids = torch.randint(-1, adapters, (rows,), generator=g, device="cuda", dtype=torch.int32)
    ids[rows // 3:] = adapters - 1 - ids[rows // 3:] % 3
    ids = ids.contiguous()
    dw = A.weight_grad(l, r, ids, adapters, out_dtype=torch.float32)
    used = torch.unique(ids[ids >= 0]).tolist()
    for a in used:
        at = torch.nonzero(ids == a).reshape(-1)
        x, y = l[at].double().t().contiguous(), r[at].double()
        want, size = torch.mm(x, y), torch.mm(x.abs(), y.abs())
        err = R.sum_error(len(at), size)
        assert bool(((dw[a].double() - want).abs() <= err + R.HALF["f32"] * (want.abs() + err)).all()), a
    rest = torch.ones(adapters, dtype=torch.bool, device="cuda")
    rest[used] = False
    assert not bool(dw[rest].any())
