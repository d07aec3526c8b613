"""GPU: dense int8 products in every width of the token tiles, against exact sums in 64 bits."""
import pytest
import torch

from tests.test_gpu_int8 import DEV, _layer, _strided, _weights

pytestmark = pytest.mark.gpu


def _tile(rows, n, sms):
    """Tokens of a dense product's tiles: by the rows, less while fewer than three quarters of the SMs would have a block."""
    bn = next(b for b, most in ((16, 16), (32, 32), (64, 64), (128, 192), (256, 1 << 40)) if rows <= most)
    while bn > 16 and -(-rows // bn) * -(-n // 128) * 4 < 3 * sms:
        bn //= 2
    return bn


@pytest.mark.parametrize("bn,rows,k", [(32, 17, 200), (32, 32, 1000), (32, 250, 96), (64, 33, 1000), (64, 64, 128), (64, 63, 2064),
                                       (64, 1000, 72), (128, 65, 400), (128, 128, 1024), (128, 191, 1000), (128, 192, 16),
                                       (128, 700, 520), (256, 193, 1000), (256, 256, 256), (256, 300, 900), (256, 513, 640),
                                       (256, 1153, 144), (256, 2500, 300)])
def test_dense_product_is_exact_in_every_tile(bn, rows, k):
    """Random rows in all tokens of a tile and weight rows that end inside a tile; the SMs of the device decide how many outputs
    it takes for tiles of bn tokens."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    tiles = -(-rows // bn)
    n = next(128 * i - 3 for i in range(1, 1000) if tiles * i * 4 >= 3 * sms)
    assert _tile(rows, n, sms) == bn
    layer = _layer()
    g = torch.Generator().manual_seed(rows + k)
    wq, ws = _weights(n, k, rows)
    xq = torch.zeros(rows, (k + 15) // 16 * 16, dtype=torch.int8)[:, :k].copy_(torch.randint(-128, 128, (rows, k), generator=g))
    xs = torch.rand(rows, generator=g) + 0.1
    y = layer.int8_matmul(_strided(xq), xs.to(DEV), _strided(wq), ws.to(DEV))
    # whole numbers below 2^53: exact in 64 bits on the device as well
    acc = (xq.to(DEV).double() @ wq.to(DEV).double().t()).float()
    assert torch.equal(y, (acc * xs.to(DEV)[:, None] * ws.to(DEV)[None, :]).to(torch.bfloat16))
    layer.close()
