"""CPU: the host-buffer forward's chunks cover the batch exactly, for chunk sizes below its edges' 128 tokens too."""
import pytest


@pytest.mark.parametrize("chunk", (1, 2, 33, 64, 100, 127, 128, 129, 200, 256, 300))
def test_small_chunks_cover_every_token_once(built_lib, chunk):
    from moe_gen_b200.layer import MoELayer
    for T in list(range(1, 600)) + [1023, 1024, 1025]:
        sizes = MoELayer.host_chunks(T, chunk)
        assert sum(sizes) == T and min(sizes) > 0, (T, chunk, sizes)
