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
