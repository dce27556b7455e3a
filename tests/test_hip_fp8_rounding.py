"""8-bit rows and weights are what their formula says, bit for bit: s = max(max|block| / 448, 2^-126), q = e4m3(x / s), with the two
divisions rounded to fp32 and the quotient to e4m3 (to nearest even).  The oracle is the CPU's own arithmetic."""
import pytest
import torch

from dsw_amd import functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F8 = torch.float8_e4m3fn
TINY = 2.0 ** -126


def _near_ties(rows, blocks, dtype, seed, size=128):
    """Blocks of many magnitudes, whose values lie on and next to the middles between two e4m3 values."""
    g = torch.Generator().manual_seed(seed)
    top = torch.ldexp(448 * (1 + torch.rand(rows, blocks, generator=g)), torch.randint(-140, 118, (rows, blocks), generator=g)).to(dtype).float()
    s = (top / 448).clamp_min(TINY)[..., None].double()
    tie = torch.ldexp(torch.randint(16, 32, (rows, blocks, size), generator=g).double(), torch.randint(-14, 4, (rows, blocks, size), generator=g))
    x = (s * tie.clamp_max(447.0)).float()
    x = (x.view(torch.int32) + torch.randint(-2, 3, x.shape, generator=g).int()).clamp_min(0).int().view(torch.float32)
    x = torch.minimum(x, top[..., None]) * (torch.randint(0, 2, x.shape, generator=g) * 2 - 1)
    x[..., 17] = top
    return x.view(rows, blocks * size).to(dtype)


def _rows(x):
    """The formula on the CPU."""
    parts = [p.float() for p in x.split(128, -1)]
    scale = [(p.abs().amax(-1) / 448.0).clamp_min(TINY) for p in parts]
    return torch.cat([(p / s[..., None]).to(F8) for p, s in zip(parts, scale)], -1), torch.stack(scale, -1)


def _same(got, q, scale, what):
    differ = int((got.scale.cpu() != scale).sum())
    assert differ == 0, "%s: %d of %d scales" % (what, differ, scale.numel())
    off = got.q.cpu().view(torch.uint8) != q.view(torch.uint8)
    assert not bool(off.any()), "%s: %d of %d values" % (what, int(off.sum()), off.numel())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,blocks,cut", [(700, 24, 0), (300, 5, 41), (3, 160, 3)])      # (the last: rows beyond the registers)
def test_rows_bit_for_bit(rows, blocks, cut, dtype):
    x = _near_ties(rows, blocks, dtype, 1)
    x = x[:, :x.shape[1] - cut].contiguous()
    _same(F.quantize_fp8(x.to(DEV)), *_rows(x), "near ties")
    x = (torch.randn(rows, blocks * 128 - cut, generator=torch.Generator().manual_seed(2)) * 7).to(dtype)
    _same(F.quantize_fp8(x.to(DEV)), *_rows(x), "normal values")
    x[1, 5], x[2, 200] = float("inf"), -float("inf")
    got = F.quantize_fp8(x.to(DEV))
    q, scale = _rows(x)
    off = (got.q.float().cpu() != q.float()) & ~(got.q.float().cpu().isnan() & q.float().isnan())
    assert torch.equal(got.scale.cpu(), scale) and not bool(off.any())                       # 0 next to an infinity, NaN in its place


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("fin,fout", [(128, 128), (300, 500), (1, 3), (129, 257), (515, 40)])
def test_weights_bit_for_bit(fin, fout, dtype):
    nb, kb = -(-fout // 128), -(-fin // 128)
    w = _near_ties(nb * kb, 1, dtype, 3, 128 * 128).view(nb, kb, 128, 128).transpose(1, 2).reshape(nb * 128, kb * 128)[:fout, :fin].contiguous()
    scale = torch.stack([torch.stack([(b.float().abs().max() / 448.0).clamp_min(TINY) for b in r.split(128, 1)]) for r in w.split(128, 0)])
    wide = scale.repeat_interleave(128, 0)[:fout].repeat_interleave(128, 1)[:, :fin]
    q = (w.float() / wide).to(F8)
    for t in (w.to(DEV).t(), w.t().contiguous().to(DEV), torch.cat([w.t(), w.t()], 1).to(DEV)[:, :fout]):
        _same(F.quantize_fp8_weight(t), q, scale, "strides %s" % (t.stride(),))
