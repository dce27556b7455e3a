"""Clipping a bucket whose parameters have no gradients yet: a norm of zero on the bucket's device, like an empty list of gradients."""
import pytest
import torch

from dsw_amd.parallel import FlatGradAllReduce, GradBucket


def _reaches_the_operator(bucket, seen, monkeypatch):
    from dsw_amd import functional

    monkeypatch.setattr(functional, "clip_grad_norm_", lambda tensors, max_norm, norm_type=2.0: seen.append((tensors, max_norm, norm_type)))
    bucket.clip_norm(2.0, 1.0)


def test_without_gradients(monkeypatch):
    bucket, seen = FlatGradAllReduce(torch.nn.Linear(4, 3).parameters()), []
    with pytest.raises(ValueError, match="max_norm"):
        bucket.clip_norm(-1.0)
    with pytest.raises(ValueError, match="norm_type"):
        bucket.clip_norm(1.0, 3.0)
    _reaches_the_operator(bucket, seen, monkeypatch)
    (tensors, max_norm, norm_type), = seen
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else tensors
    assert len(tensors) == 1 and tensors[0].numel() == 0 and tensors[0].device == bucket.bucket.device and (max_norm, norm_type) == (2.0, 1.0)


@pytest.mark.gpu
def test_without_gradients_on_the_gpu():
    lin = torch.nn.Linear(4, 3).to("cuda")
    bucket = GradBucket(lin.parameters(), attach=False)
    for p in (2.0, 1.0, float("inf")):
        n = bucket.clip_norm(1.0, p)
        assert n.is_cuda and n.dim() == 0 and n.dtype == torch.float32 and float(n) == 0.0
    assert all(q.grad is None for q in lin.parameters())
    lin.weight.grad = torch.full_like(lin.weight, 2.0)                   # some have one
    assert float(bucket.clip_norm(1.0, float("inf"))) == 2.0 and lin.bias.grad is None
    assert float((lin.weight.grad - 1.0).abs().max()) <= 2.0 ** -20       # 1 / (2 + 1e-6)
