"""The residual branch's 8-bit path serves the weight that the layer has now, or raises (host logic: plain stand-ins for the quantiser
and the product, so these run on the CPU)."""
import copy
import io

import pytest
import torch
import torch.nn.utils.parametrize  # noqa: F401

from dsw_amd import functional as F
from modules import my_models_graph as M


@pytest.fixture()
def stand_ins(monkeypatch):
    """The quantised weight is a copy of its values, the product an ordinary one in their precision."""
    made = []

    def quantize(weight):
        made.append(weight)
        return F.Fp8Weight(weight.detach().t().clone(), torch.ones(1, 1))

    monkeypatch.setattr(M.dsw_functional, "quantize_fp8_weight", quantize)
    monkeypatch.setattr(M.dsw_functional, "dense_mix_fp8", lambda x, w, bias=None: x @ w.q.t() + bias)
    return made


def _served(lin, x):
    """What the layer answers under no_grad: a tensor, or None where it raises that the weight has changed."""
    with torch.no_grad():
        try:
            return lin(x)
        except RuntimeError as exc:
            assert "has changed" in str(exc)
            return None


def _right(lin, x):
    """The layer's answer is the present weight's, or it raises."""
    y = _served(lin, x)
    return y is None or torch.equal(y, x @ lin.weight.detach().t() + lin.bias.detach())


def test_another_tensor_in_the_weights_place(stand_ins):
    """Samples of an ensemble are plain tensors assigned by attribute, each of them at version 0."""
    x = torch.randn(5, 6)
    lin = M._NodeLinear(6, 4)
    del lin._parameters["weight"]
    samples = [torch.randn(4, 6) for _ in range(2)]
    lin.weight = samples[0]
    lin.serve_fp8()
    assert _served(lin, x) is not None and _right(lin, x)
    lin.weight = samples[1]
    assert samples[0]._version == samples[1]._version and _right(lin, x)
    lin.serve_fp8()
    assert _served(lin, x) is not None and _right(lin, x)
    del lin.weight                              # the tensor that it was made from dies, another one may take its place in memory
    samples.clear()
    lin.weight = torch.randn(4, 6)
    assert _right(lin, x)


def test_states_that_are_assigned(stand_ins):
    x = torch.randn(5, 6)
    lin = M._NodeLinear(6, 4).serve_fp8()
    states = [{"weight": torch.randn(4, 6), "bias": torch.randn(4)} for _ in range(2)]
    for state in states:
        lin.load_state_dict(state, assign=True)
        assert _right(lin, x)
        lin.serve_fp8()
        assert _served(lin, x) is not None and _right(lin, x)


def test_a_parametrised_weight(stand_ins):
    """Its layer has another tensor each time it is asked for the weight: what is served follows the parameters below it."""
    class Twice(torch.nn.Module):
        def forward(self, w):
            return 2 * w

    x = torch.randn(5, 6)
    lin = M._NodeLinear(6, 4)
    torch.nn.utils.parametrize.register_parametrization(lin, "weight", Twice())
    lin.serve_fp8()
    for _ in range(2):
        assert _served(lin, x) is not None and _right(lin, x)
        lin.parametrizations.weight.original.data.add_(1.0)


def test_copies_start_in_their_own_precision(stand_ins):
    """A copy has a weight of its own: it does not inherit the switch, and copying or pickling a served layer works."""
    x = torch.randn(5, 6)
    lin = M._NodeLinear(6, 4).serve_fp8()
    stand_ins.clear()
    twin = copy.deepcopy(lin)
    buf = io.BytesIO()
    torch.save(lin, buf)
    buf.seek(0)
    for other in (twin, torch.load(buf, weights_only=False)):
        assert other._fp8 is None and torch.equal(other.weight, lin.weight)
        with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU fallback"):        # the layer's ordinary path
            other(x)
    assert not stand_ins and _right(lin, x)


def test_writes_that_autograd_does_not_see(stand_ins):
    """Writes through ``weight.data`` (a replayed optimizer step is one, too) leave the version as it is: what is served is the
    weight as it is now."""
    x = torch.randn(5, 6)
    lin = M._NodeLinear(6, 4).serve_fp8()
    before = _served(lin, x)
    lin.weight.data.mul_(3.0)
    assert _right(lin, x) and not torch.equal(_served(lin, x), before)
    with torch.no_grad():
        lin.weight.add_(1.0)
    assert _served(lin, x) is None                                # autograd's own count: raises, as promised
    assert _right(lin.serve_fp8(), x) and _served(lin, x) is not None


def _block(cin, widths):
    from dsw_amd import sphere
    from modules.layers import prepare_torch_laplacian

    lap = prepare_torch_laplacian(sphere.SphereHealpix(4, nest=True, k=8).L, lmax=1.9)
    opts = dict(kernel_size=3, conv_type="graph", bias=True, batch_norm=False, batch_norm_before_activation=False,
                activation=True, activation_fun="relu", periodic_padding=True, lonlat_ratio=None)
    return M.ResBlock(cin, widths, laplacian=lap, convblock_kwargs=opts)


def test_a_block_with_a_fused_tail_serves_its_branch(stand_ins, oracle_backend, monkeypatch):
    """Where the last convolution would take the block's tail and read the branch's weight itself, the switch decides."""
    monkeypatch.setattr(M.ResBlock, "fuse_tail", True)
    block, x = _block(6, (12, 10)), torch.randn(2, 192, 6)
    with torch.no_grad():
        plain = block(x)
        assert block._fusable_tail(x) and M.serve_fp8(block) == 1
        stand_ins.clear()
        y = block(x)
        assert len(stand_ins) == 1 and float((y - plain).abs().max()) <= 1e-5 * float(plain.abs().max())
        block.res_connection.weight.add_(1.0)
        with pytest.raises(RuntimeError, match="has changed"):
            block(x)
        M.serve_fp8(block)
    assert block._fusable_tail(x)                               # with gradients the layer is what it was
    stand_ins.clear()
    block(x.requires_grad_()).sum().backward()
    assert not stand_ins and block.res_connection.weight.grad is not None


@pytest.mark.gpu
@pytest.mark.parametrize("fuse_tail", [False, True])
def test_every_served_branch_takes_the_8_bit_product(fuse_tail, monkeypatch):
    """One 8-bit product for each branch that serve_fp8 counts, as the library's launch trace sees them."""
    from dsw_amd import _native

    monkeypatch.setattr(M.ResBlock, "fuse_tail", fuse_tail)
    blocks = [_block(18, (64, 128)), _block(128, (64, 32)), _block(32, (32,)), _block(32, 2)]
    model = torch.nn.Sequential(*blocks).to("cuda").eval()
    x = torch.randn(2, 192, 18, device="cuda")
    with torch.no_grad():
        model(x)
        found = M.serve_fp8(model)
        with _native.LaunchTrace() as trace:
            model(x)
            torch.cuda.synchronize()
    assert found == 3 and [r[1:4] for r in trace.intervals if r[0] == "fp8_mix"] == [(384, 18, 128), (384, 128, 32), (384, 32, 2)]


def _alike(a, b):
    return a.dtype == b.dtype and a.shape == b.shape and torch.equal(a, b)


@pytest.mark.gpu
def test_a_replayed_update_reaches_the_served_weight():
    """serve_fp8 - an optimizer step that is replayed from a graph - inference: the new weight's values."""
    torch.manual_seed(0)
    lin = M._NodeLinear(200, 72).to("cuda")
    x, new = torch.randn(90, 200, device="cuda"), torch.randn(72, 200, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.no_grad():
        lin.weight.add_(new)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    update = torch.cuda.CUDAGraph()
    with torch.cuda.graph(update), torch.no_grad():
        lin.weight.add_(new)
    lin.serve_fp8()
    for _ in range(3):
        update.replay()
        with torch.no_grad():
            y = lin(x)
            want = F.dense_mix_fp8(x, F.quantize_fp8_weight(lin.weight.t()), lin.bias)
        torch.cuda.synchronize()
        assert _alike(y, want)


@pytest.mark.gpu
def test_captured_inference_follows_the_weight():
    """A captured inference graph answers with the weight at each replay, whatever is done with the switch in between."""
    torch.manual_seed(0)
    lin = M._NodeLinear(130, 72).to("cuda").serve_fp8()
    x = torch.randn(90, 130, device="cuda")
    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            lin(x)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = lin(x)
        for step in range(4):
            lin.weight.mul_(-1.5)
            if step % 2 == 0:
                lin.serve_fp8(step == 0)                      # again, and off: the graph's own memory is not theirs
            trash = [torch.full((72, 130), 7, dtype=torch.uint8, device="cuda") for _ in range(8)]
            graph.replay()
            torch.cuda.synchronize()
            assert _alike(y, F.dense_mix_fp8(x, F.quantize_fp8_weight(lin.weight.t()), lin.bias))
            assert all(bool((t == 7).all()) for t in trash)
