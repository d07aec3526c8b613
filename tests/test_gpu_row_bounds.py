"""GPU: buffers of fewer rows than the plan's table names.  The picks whose rows do not exist are left out of every movement and of
its gradient, and nothing outside the buffers is read or written."""
import itertools

import pytest
import torch

from tests.test_gpu_grad import DEV, _setup

pytestmark = pytest.mark.gpu
T, E, k, H = 70, 8, 2, 512


def _clipped(dst, n):
    return torch.where(dst < n, dst, torch.full_like(dst, -1))


def _buffers(seed):
    layer, idx, counts, pad, dst, rows, live = _setup(T, E, k, H)
    g = torch.Generator().manual_seed(seed)
    some = int(dst.float().median())                      # about half the picks lie below
    assert 0 < some < int(dst.max())
    return layer, idx, counts, pad, dst, rows, some, g


@pytest.mark.parametrize("mode,with_shared", list(itertools.product((0, 1, 2), (False, True))))
def test_return_of_rows_that_are_not_there(mode, with_shared):
    from moe_gen_b200 import combine_rows
    layer, idx, counts, pad, dst, rows, live = _setup(T, E, k, H, combine=mode)
    g = torch.Generator().manual_seed(mode)
    big = torch.randn(rows, H, generator=g).to(torch.bfloat16).to(DEV)
    w = torch.rand(T, k, generator=g).to(DEV)
    sh = torch.randn(T, H, generator=g).to(torch.bfloat16).to(DEV) if with_shared else None
    gy = torch.randn(T, H, generator=g).to(torch.bfloat16).to(DEV)
    for n in (0, 1, int(dst.float().median()), int(dst.max()), int(dst.max()) + 1):
        big[n:] = float("nan")                            # what a read behind the buffer would bring in
        out = big[:n]
        y = combine_rows(layer, out, dst, idx, w, counts, pad, sh)
        cut = _clipped(dst, n)
        want = layer.combine(torch.nan_to_num(big), cut, idx, w, sh)
        assert torch.equal(y, want)
        leaves = [out.clone().requires_grad_(True), w.clone().requires_grad_(True)]
        gr, gw = torch.autograd.grad(combine_rows(layer, leaves[0], dst, idx, leaves[1], counts, pad), leaves, gy)
        assert not gw[cut < 0].any()
        wr = w.to(torch.bfloat16).float() if mode else w
        t, j = (cut >= 0).nonzero(as_tuple=True)
        assert torch.equal(gr[cut[t, j].long()], (gy[t].float() * wr[t, j, None]).to(torch.bfloat16))
        big = torch.randn(rows, H, generator=g).to(torch.bfloat16).to(DEV)
    layer.close()


def test_sort_into_too_few_rows_and_its_gradient():
    from moe_gen_b200 import sort_rows
    layer, idx, counts, pad, dst, rows, some, g = _buffers(3)
    x = torch.randn(T, H, generator=g).to(torch.bfloat16).to(DEV)
    full = layer.permute_rows(x, dst, rows)
    for n in (1, some, int(dst.max())):
        leaf = x.clone().requires_grad_(True)
        perm = sort_rows(layer, leaf, dst, n, counts, pad)
        assert torch.equal(perm, full[:n]) and torch.equal(layer.permute_rows(x, dst, n), full[:n])
        gr = torch.randn(rows, H, generator=g).to(torch.bfloat16).to(DEV)
        want = layer.permute_rows_grad(gr, _clipped(dst, n))
        gr[n:] = float("nan")
        assert torch.equal(torch.autograd.grad(perm, leaf, gr[:n])[0], want)
        assert torch.equal(layer.permute_rows_grad(gr[:n], dst), want)
    assert not layer.permute_rows_grad(full[:0], dst).any()
    layer.close()


def test_quantised_rows_into_too_few_rows():
    layer, idx, counts, pad, dst, rows, some, g = _buffers(4)
    x = torch.randn(T, H, generator=g).to(torch.bfloat16).to(DEV)
    q, s = layer.quantize_rows(x)
    fq, fs = layer.permute_rows_int8(q, s, dst, rows)
    for n in (1, some):
        pq, ps = layer.permute_rows_int8(q, s, dst, n)
        at = dst[dst < n].long()
        assert pq.shape == (n, H) and ps.shape == (n,) and torch.equal(pq[at], fq[at]) and torch.equal(ps[at], fs[at])
    layer.close()


@pytest.mark.parametrize("int8", (False, True))
def test_nothing_behind_the_named_rows_is_written(int8):
    from moe_gen_b200 import lib as L
    layer, idx, counts, pad, dst, rows, some, g = _buffers(5)
    x = torch.randn(T, H, generator=g).to(torch.bfloat16).to(DEV)
    q, s = layer.quantize_rows(x)
    src, ref = (q, layer.permute_rows_int8(q, s, dst, rows)[0]) if int8 else (x, layer.permute_rows(x, dst, rows))
    buf = torch.full((rows, H), 77, dtype=src.dtype, device=DEV)
    sc = torch.full((rows,), 77.0, device=DEV)
    L.check(layer.lib.mg_permute_rows_bounded(layer._h, src.data_ptr(), s.data_ptr() if int8 else None, dst.data_ptr(), T, some,
                                              buf.data_ptr(), sc.data_ptr() if int8 else None, layer._stream()))
    at = dst[dst < some].long()
    assert torch.equal(buf[at], ref[at]) and bool((buf[some:] == 77).all()) and bool((sc[some:] == 77).all())
    with pytest.raises(L.MoeGenError):                    # scales on one side only
        L.check(layer.lib.mg_permute_rows_bounded(layer._h, src.data_ptr(), s.data_ptr(), dst.data_ptr(), T, some, buf.data_ptr(), None,
                                                  layer._stream()))
    layer.close()


def test_tables_of_other_tokens_are_refused():
    layer, idx, counts, pad, dst, rows, some, g = _buffers(6)
    x = torch.zeros(T, H, dtype=torch.bfloat16, device=DEV)
    for bad in (lambda: layer.permute_rows(x, dst[:5], rows), lambda: layer.permute_rows(x, dst.long(), rows),
                lambda: layer.permute_rows(x[:, :256].contiguous(), dst, rows), lambda: layer.permute_rows(x, dst[:, :1], rows)):
        with pytest.raises(ValueError):
            bad()
    layer.close()
