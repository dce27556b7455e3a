"""Row norm, every arrangement of threads and registers, with more rows than a launch has workgroups: the loops over rows, their
look-ahead and the column sums over several rows of a workgroup, against 64 bits (plain torch operations in float64 on the GPU).

Bounds (u = 2^-24, r = half a step of the output type): a row's square sum has n <= 72 + C / 256 roundings in any one path (a lane's
chain, the joins); y then half of that (square root) and 6 more; a column sum of dw has at most rows / 512 terms in a thread's chain
(512 workgroups), 16 joins in the workgroup, 8 + 2 + 16 over the workgroups' partial sums."""
import pytest
import torch

from dsw_amd import functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
EPS = 1e-5
# channels in 16-byte vectors (8 bf16 or 4 fp32 channels each) and rows: 16, 32, 64 lanes a row; 2, 4 vectors a lane; a workgroup a row
# with 2, 4, 8 vectors a thread; longer than the registers
SHAPES = [(16, 70001), (31, 33001), (62, 17001), (125, 17001), (255, 17001), (500, 8301), (1023, 8301), (2000, 8301), (2500, 1301)]


def _within(got, want, tol, what):
    worst = ((got.detach().double() - want).abs() / tol.clamp_min(1e-300)).max()
    assert float(worst) <= 1.0, "%s: %.3g of the bound" % (what, float(worst))


def _inputs(rows, C, dtype, count):
    g = torch.Generator(device=DEV).manual_seed(rows + C)
    made = [(torch.randn(rows, C, generator=g, device=DEV) * (1 if i else 2)).to(dtype) for i in range(count)]
    return made, (1 + 0.3 * torch.randn(C, generator=g, device=DEV)).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("vectors,rows", SHAPES)
def test_forward_and_backward(vectors, rows, residual, dtype):
    C = vectors * (8 if dtype == torch.bfloat16 else 4) - (3 if vectors % 2 else 0)
    (x, r, dy, dh), w = _inputs(rows, C, dtype, 4)
    leaves = [t.requires_grad_() for t in ((x, r, w) if residual else (x, w))]
    if residual:
        y, h = F.rms_norm_residual(x, r, w, EPS)
        dx, dr, dw = torch.autograd.grad((y, h), leaves, (dy, dh))
        assert torch.equal(dx, dr)
    else:
        y, h = F.rms_norm(x, w, EPS), None
        dx, dw = torch.autograd.grad(y, leaves, dy)
    x, r, w = (t.detach() for t in (x, r, w))
    n = 72 + C / 256
    h64 = x.double() + r.double() if residual else x.double()
    rstd = (h64.square().mean(-1, keepdim=True) + EPS).rsqrt()
    xhat = h64 * rstd
    if residual:
        _within(h, h64, (HALF[dtype] + 2 * U) * h64.abs(), "h")
    del h64
    want = xhat * w.double()
    _within(y, want, (HALF[dtype] + (n / 2 + 6) * U) * want.abs(), "y")
    terms = dy.double() * xhat
    want, mag = terms.sum(0), terms.abs().sum(0)
    _within(dw, want, (HALF[dtype] + U) * want.abs() + (n / 2 + 6 + rows / 512 + 48) * U * mag, "dw")
    gw = dy.double() * w.double()
    terms = gw * xhat
    a, mag = terms.mean(-1, keepdim=True), terms.abs().mean(-1, keepdim=True)
    want = rstd * (gw - xhat * a)
    tol = 2 * n * U * rstd * (gw.abs() + xhat.abs() * mag)
    if residual:
        want += dh.double()
        tol += 2 * U * dh.double().abs()
    _within(dx, want, tol + (HALF[dtype] + 2 * U) * want.abs(), "dx")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vectors,rows", [(s, n if n < 70000 else 2 * n) for s, n in SHAPES])
def test_8_bit_output(vectors, rows, dtype):
    """Scales within the computing error and 2 roundings, values within half a step of e4m3 (2^-4, 2^-10 of the scale at the lower end)."""
    C = vectors * (8 if dtype == torch.bfloat16 else 4) - (3 if vectors % 2 else 0)
    (x, r), w = _inputs(rows, C, dtype, 2)
    got, h = F.rms_norm_fp8(x, w, residual=r, eps=EPS)
    rel = (36 + C / 512 + 6) * U
    h64 = x.double() + r.double()
    _within(h, h64, (HALF[dtype] + 2 * U) * h64.abs(), "h")
    y64 = h64 * (h64.square().mean(-1, keepdim=True) + EPS).rsqrt() * w.double()
    for b, part in enumerate(y64.split(128, -1)):
        scale = (part.abs().amax(-1) / 448).clamp_min(2.0 ** -126)
        mine = got.scale[:, b].double()
        _within(mine, scale, scale * (rel + 3 * U), "scale of block %d" % b)
        q = got.q[:, 128 * b:128 * b + part.shape[1]].float().double() * mine[:, None]
        _within(q, part, torch.maximum(2.0 ** -4 * part.abs(), 2.0 ** -10 * mine[:, None]) + (rel + 6 * U) * part.abs(), "q of block %d" % b)


def test_more_rows_than_a_grid_of_whole_workgroups():
    """2^20 workgroups of a row each walk on: forward of rows that a workgroup shares, and their 8-bit form."""
    rows, C = (1 << 20) + 777, 2064
    g = torch.Generator(device=DEV).manual_seed(7)
    x = torch.empty(rows, C, dtype=torch.bfloat16, device=DEV).normal_(generator=g)
    w = (1 + 0.3 * torch.randn(C, generator=g, device=DEV)).bfloat16()
    y, q = F.rms_norm(x, w, EPS), F.rms_norm_fp8(x, w, eps=EPS)[0]
    n = 72 + C / 256
    for at in range(0, rows, 1 << 17):
        part = slice(at, min(rows, at + (1 << 17)))
        h64 = x[part].double()
        want = h64 * (h64.square().mean(-1, keepdim=True) + EPS).rsqrt() * w.double()
        _within(y[part], want, (HALF[torch.bfloat16] + (n / 2 + 6) * U) * want.abs(), "y from row %d" % at)
        s = q.scale[part].double().repeat_interleave(128, -1)[:, :C]
        _within(q.q[part].float() * s, want, torch.maximum(2.0 ** -4 * want.abs(), 2.0 ** -10 * s) + (n / 2 + 12) * U * want.abs(), "q from row %d" % at)
