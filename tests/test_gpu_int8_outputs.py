"""GPU: int8 products of nearly 2^31 outputs."""
import pytest
import torch

from tests.test_gpu_int8 import DEV, _layer, product, quantise, same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,n", [(1, (1 << 30) + 8), (2, (1 << 31) - 520)])
def test_first_and_last_outputs(rows, n):
    free, _ = torch.cuda.mem_get_info()
    if free < 80 << 30:
        pytest.skip("needs 80 GB")
    layer, k, ends = _layer(), 16, 5000
    g = torch.Generator().manual_seed(rows)
    wq = torch.zeros(n, k, dtype=torch.int8, device=DEV)
    ws = torch.ones(n, device=DEV)
    first, last = (torch.randint(-128, 128, (ends, k), generator=g, dtype=torch.int8) for _ in range(2))
    wq[:ends], wq[-ends:] = first.to(DEV), last.to(DEV)
    x = torch.randn(rows, k, generator=g).to(torch.bfloat16)
    guard = torch.full((rows + 2, n), 7.0, dtype=torch.bfloat16, device=DEV)
    y = layer.int8_linear(x.to(DEV), wq, ws, out=guard[1:rows + 1])
    q, s = quantise(x)
    assert same(y[:, :ends].cpu(), product(q, s, first, torch.ones(ends))) and same(y[:, -ends:].cpu(), product(q, s, last, torch.ones(ends)))
    assert all(not c.any() for r in y for c in r[ends:-ends].split(1 << 28))
    assert all(bool((c == 7.0).all()) for r in (guard[0], guard[-1]) for c in r.split(1 << 28))
    layer.close()
    del wq, ws, guard, y
    torch.cuda.empty_cache()
