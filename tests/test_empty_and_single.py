"""Row norm and 8-bit product: no rows, a single output, whatever the strides say of an axis of length one."""
import pytest
import torch

from dsw_amd import _native, functional as F

DEV = "cuda:0"
F8 = torch.float8_e4m3fn


def test_backward_entry_without_rows():
    """No rows, dW not asked for: nothing to do, and the pointers of empty tensors are null."""
    lib = _native.load()
    p = 4096
    assert lib.dsw_rmsnorm_bwd(None, None, None, 8, None, 0, p, None, None, None, None, 0, 0, 8, 0, None) == 0
    assert lib.dsw_rmsnorm_bwd(p, None, p, 8, None, 0, p, p, None, None, None, 0, 4, 8, 0, None) == -1        # with rows: a result is


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lead", [(0,), (3, 0), (0, 5)])
def test_norm_without_rows(lead, dtype):
    """Every combination of inputs that want a gradient."""
    for want in range(1, 8):
        x, r, w = (torch.zeros(s, dtype=dtype, device=DEV, requires_grad=bool(want >> i & 1)) for i, s in enumerate(((*lead, 36), (*lead, 36), (36,))))
        y, h = F.rms_norm_residual(x, r, w)
        (y.sum() + h.sum()).backward()
        for t in (x, r, w):
            assert (t.grad is not None) == t.requires_grad and (t.grad is None or (t.grad.shape == t.shape and bool((t.grad == 0).all())))
        if want & 5:
            x.grad = w.grad = None
            F.rms_norm(x, w).sum().backward()
            for t in (x, w):
                assert (t.grad is not None) == t.requires_grad and (t.grad is None or (t.grad.shape == t.shape and bool((t.grad == 0).all())))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 40, 300])
def test_product_with_one_output(rows):
    """One row of weights: the stride between rows means nothing, however large or small it is."""
    K = 272
    g = torch.Generator().manual_seed(0)
    xq = (torch.randn(rows, K, generator=g) * 60).clamp(-448, 448).to(F8).to(DEV)
    wq = (torch.randn(1, K, generator=g) * 60).clamp(-448, 448).to(F8).to(DEV)
    xs, ws = torch.rand(rows, 3, generator=g).to(DEV), torch.rand(1, 3, generator=g).to(DEV)
    want = F.dense_mix_fp8(F.Fp8Rows(xq, xs), F.Fp8Weight(wq, ws), dtype=torch.float32)
    for stride in ((1 << 23) + 16, (1 << 23) + 5, 1 << 40, 7, 0):
        odd = wq.as_strided((1, K), (stride, 1))
        assert torch.equal(F.dense_mix_fp8(F.Fp8Rows(xq, xs), F.Fp8Weight(odd, ws), dtype=torch.float32), want), stride
    one = F.dense_mix_fp8(F.Fp8Rows(xq[:1].as_strided((1, K), (1 << 40, 1)), xs[:1]), F.Fp8Weight(wq, ws), dtype=torch.float32)
    assert torch.equal(one, F.dense_mix_fp8(F.Fp8Rows(xq[:1], xs[:1]), F.Fp8Weight(wq, ws), dtype=torch.float32))
    x1, w1 = xq[:, :1], wq.t()[:5, :1]                                    # one channel: neither has its stride
    got = F.dense_mix_fp8(F.Fp8Rows(x1, xs[:, :1]), F.Fp8Weight(w1, ws[:, :1]), dtype=torch.float32)
    assert torch.equal(got, F.dense_mix_fp8(F.Fp8Rows(x1.contiguous(), xs[:, :1].contiguous()), F.Fp8Weight(w1.contiguous(), ws[:, :1].contiguous()), dtype=torch.float32))
