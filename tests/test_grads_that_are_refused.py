"""What the row norm, the 8-bit product and the gradient norm cannot differentiate raises instead of losing a derivative (CPU: the
checks come before the device's)."""
import pytest
import torch

from dsw_amd import functional as F

F8 = torch.float8_e4m3fn
passed = lambda: pytest.raises(RuntimeError, match="no CPU fallback")  # noqa: E731  (every check of the arguments passed)
refused = lambda: pytest.raises(RuntimeError, match="no_grad|detach")  # noqa: E731


def test_gradient_norms_have_no_backward():
    leaf = torch.randn(5, requires_grad=True)
    (grad,) = torch.autograd.grad(leaf.square().sum(), leaf, create_graph=True)
    plain = torch.randn(5)
    for tensors in ([leaf], [grad], [plain, grad]):
        with refused():
            F.grad_norm(tensors)
        with refused():
            F.clip_grad_norm_(tensors, 1.0)
        with torch.no_grad():
            with passed():
                F.grad_norm(tensors)
            with passed():
                F.clip_grad_norm_(tensors, 1.0)
        with passed():
            F.grad_norm([t.detach() for t in tensors])
    with refused():
        F.clip_grad_norm_([plain], 1.0, out=[leaf])
    with passed():
        F.clip_grad_norm_([plain], 1.0, out=[torch.empty(5)])


def test_clipping_a_bucket_does_not_mind_parameters():
    """The bucket's own call: gradients of parameters, with autograd on around it."""
    from dsw_amd.parallel import FlatGradAllReduce, GradBucket

    lin = torch.nn.Linear(4, 3)
    for bucket in (GradBucket(lin.parameters()), FlatGradAllReduce(lin.parameters())):
        if bucket.attached:
            bucket.zero()
        lin(torch.randn(2, 4)).sum().backward()
        with passed():
            bucket.clip_norm(1.0)
    for p in lin.parameters():                        # gradients with a graph of their own are clipped as torch clips them: under no_grad
        p.grad = None
    lin(torch.randn(2, 4)).square().sum().backward(create_graph=True)
    assert lin.weight.grad.requires_grad
    with passed():
        bucket.clip_norm(1.0)


def test_forward_mode_derivatives_are_refused():
    """A tangent of any operand, with and without no_grad: a result without one would read as a derivative of zero."""
    import torch.autograd.forward_ad as fwd

    x, w, r, bias = torch.randn(4, 8), torch.ones(8), torch.randn(4, 8), torch.zeros(3)
    q8 = F.Fp8Rows(torch.zeros(4, 8, dtype=F8), torch.ones(4, 1))
    w8 = F.Fp8Weight(torch.zeros(3, 8, dtype=F8), torch.ones(1, 1))
    calls = [(lambda d: F.rms_norm(d, w), x), (lambda d: F.rms_norm(x, d), w), (lambda d: F.rms_norm_residual(d, r, w), x),
             (lambda d: F.rms_norm_residual(x, d, w), r), (lambda d: F.rms_norm_residual(x, r, d), w),
             (lambda d: F.rms_norm_fp8(d, w), x), (lambda d: F.rms_norm_fp8(x, d), w), (lambda d: F.rms_norm_fp8(x, w, residual=d), r),
             (lambda d: F.quantize_fp8(d), x), (lambda d: F.quantize_fp8_weight(d), x), (lambda d: F.dense_mix_fp8(d, w8), x),
             (lambda d: F.dense_mix_fp8(q8, w8, d, dtype=torch.float32), bias),
             (lambda d: F.dense_mix_fp8(F.Fp8Rows(q8.q, d), w8), q8.scale), (lambda d: F.dense_mix_fp8(q8, F.Fp8Weight(w8.q, d)), w8.scale),
             (lambda d: F.grad_norm([x, d]), r), (lambda d: F.clip_grad_norm_([x, d], 1.0), r),
             (lambda d: F.clip_grad_norm_([x], 1.0, out=[d]), r)]
    for i, (call, operand) in enumerate(calls):
        with passed():
            call(operand)
        for grad in (True, False):
            with fwd.dual_level(), torch.set_grad_enabled(grad):
                dual = fwd.make_dual(operand, torch.ones_like(operand))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call(dual)
                with passed():
                    call(fwd.unpack_dual(dual).primal)


@pytest.mark.gpu
def test_function_transforms_are_refused():
    """Wrapped tensors of torch.func have no memory that a kernel could read: they raise."""
    x, w = torch.randn(4, 8, device="cuda"), torch.ones(8, device="cuda")
    w8 = F.quantize_fp8_weight(torch.randn(8, 3, device="cuda"))
    for call in (lambda t: F.rms_norm(t, w).sum(), lambda t: F.rms_norm_residual(t, t, w)[1].sum(), lambda t: F.grad_norm([t]),
                 lambda t: F.dense_mix_fp8(t, w8).sum(), lambda t: F.rms_norm_fp8(t, w)[0].scale.sum()):
        for transform in (lambda f: torch.func.grad(f)(x), lambda f: torch.func.jvp(f, (x,), (x,)), lambda f: torch.func.vmap(f)(x[None])):
            with pytest.raises(RuntimeError):
                transform(call)
    torch.cuda.synchronize()
