"""Row norm, 8-bit channel mix, gradient clipping: what the host refuses, before anything is launched (CPU)."""
import ctypes
import math

import numpy as np
import pytest
import torch

from dsw_amd import _native, functional as F

F8 = torch.float8_e4m3fn


# a call that passes every check of its arguments ends at the device of its tensors
passed = lambda: pytest.raises(RuntimeError, match="no CPU fallback")  # noqa: E731


def test_cpu_tensors_are_refused():
    x, w = torch.randn(4, 8), torch.ones(8)
    for call in (lambda: F.rms_norm(x, w), lambda: F.rms_norm_residual(x, x, w), lambda: F.rms_norm_fp8(x, w), lambda: F.quantize_fp8(x),
                 lambda: F.quantize_fp8_weight(x), lambda: F.grad_norm([x]), lambda: F.clip_grad_norm_([x], 1.0),
                 lambda: F.dense_mix_fp8(F.Fp8Rows(torch.zeros(4, 8, dtype=F8), torch.ones(4, 1)),
                                         F.Fp8Weight(torch.zeros(3, 8, dtype=F8), torch.ones(1, 1)))):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


def test_norm_refusals():
    x, w = torch.randn(4, 8), torch.ones(8)
    with pytest.raises(ValueError):
        F.rms_norm(x, torch.ones(7))
    with pytest.raises(ValueError):
        F.rms_norm(x, torch.ones(1, 8))
    with pytest.raises(ValueError):
        F.rms_norm(torch.randn(4, 0), torch.ones(0))
    with pytest.raises(ValueError):
        F.rms_norm(torch.tensor(1.0), torch.ones(1))
    for eps in (-1e-6, math.nan, math.inf):
        with pytest.raises(ValueError, match="eps"):
            F.rms_norm(x, w, eps)
    with pytest.raises(ValueError):
        F.rms_norm_residual(x, torch.randn(1, 8), w)
    with pytest.raises(TypeError, match="mixed"):
        F.rms_norm(x, w.bfloat16())
    with pytest.raises(TypeError, match="mixed"):
        F.rms_norm_residual(x, x.bfloat16(), w)
    with pytest.raises(TypeError, match="unsupported"):
        F.rms_norm(x.double(), w.double())
    with pytest.raises(TypeError, match="unsupported"):
        F.quantize_fp8(x.half())
    with pytest.raises(RuntimeError, match="no_grad"):
        F.rms_norm_fp8(x, torch.nn.Parameter(w))
    with passed():
        with torch.no_grad():
            F.rms_norm_fp8(x, torch.nn.Parameter(w))
    with passed():
        F.rms_norm_residual(x, x, w)


def test_product_refusals():
    rows = F.Fp8Rows(torch.zeros(4, 300, dtype=F8), torch.ones(4, 3))
    weight = F.Fp8Weight(torch.zeros(130, 300, dtype=F8), torch.ones(2, 3))
    with passed():
        F.dense_mix_fp8(rows, weight)
    with passed():
        F.dense_mix_fp8(rows, weight, torch.zeros(130, dtype=torch.bfloat16))
    with pytest.raises(TypeError):
        F.dense_mix_fp8(rows, weight.q)
    with pytest.raises(TypeError):
        F.dense_mix_fp8((rows.q, rows.scale), weight)
    with pytest.raises(TypeError, match="float8"):
        F.dense_mix_fp8(F.Fp8Rows(rows.q.view(torch.uint8), rows.scale), weight)
    with pytest.raises(TypeError, match="scales"):
        F.dense_mix_fp8(F.Fp8Rows(rows.q, rows.scale.double()), weight)
    with pytest.raises(TypeError, match="unsupported"):
        F.dense_mix_fp8(rows, weight, dtype=torch.float16)
    with pytest.raises(TypeError, match="mixed"):
        F.dense_mix_fp8(rows, weight, torch.zeros(130))
    for bad in (F.Fp8Rows(rows.q[:, :299], rows.scale), F.Fp8Rows(rows.q, rows.scale[:, :2]), F.Fp8Rows(rows.q, rows.scale[:3])):
        with pytest.raises(ValueError):
            F.dense_mix_fp8(bad, weight)
    with pytest.raises(ValueError):
        F.dense_mix_fp8(rows, F.Fp8Weight(weight.q, weight.scale.t()))
    with pytest.raises(ValueError):
        F.dense_mix_fp8(rows, weight, torch.zeros(131, dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        F.dense_mix_fp8(torch.randn(4, 299), weight)
    with pytest.raises(RuntimeError, match="no_grad"):
        F.dense_mix_fp8(torch.randn(4, 300, requires_grad=True), weight)


def test_clip_refusals():
    g = [torch.randn(5), torch.randn(2, 3)]
    with passed():
        F.clip_grad_norm_(g, 1.0)
    with pytest.raises(ValueError):
        F.clip_grad_norm_([], 1.0)
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            F.clip_grad_norm_(g, bad)
    for p in (0.0, 3.0, -math.inf, math.nan):
        with pytest.raises(ValueError, match="norm_type"):
            F.grad_norm(g, p)
    with pytest.raises(TypeError, match="unsupported"):
        F.grad_norm([g[0].double()])
    with pytest.raises(ValueError, match="out"):
        F.clip_grad_norm_(g, 1.0, out=g[:1])
    with pytest.raises(ValueError, match="out"):
        F.clip_grad_norm_(g, 1.0, out=[g[0], g[1].t()])
    with pytest.raises(ValueError, match="out"):
        F.clip_grad_norm_(g, 1.0, out=[g[0], g[1].bfloat16()])
    with pytest.raises(ValueError, match="dense"):
        F.clip_grad_norm_([torch.randn(4, 4)[:, ::2]], 1.0)


def test_c_entries_refuse_before_they_launch():
    """Codes of the C entries for arguments that no kernel may see; nothing here is a device pointer."""
    lib = _native.load()
    p = 4096
    assert lib.dsw_rmsnorm_fwd(p, 8, None, 0, p, p, None, None, 4, 8, 1e-6, 7, None) == -2
    assert lib.dsw_rmsnorm_fwd(p, 7, None, 0, p, p, None, None, 4, 8, 1e-6, 0, None) == -1          # rows overlap
    assert lib.dsw_rmsnorm_fwd(p, 8, p, 8, p, p, None, None, 4, 8, 1e-6, 0, None) == -1              # a residual without h
    assert lib.dsw_rmsnorm_fwd(p, 8, None, 0, None, p, None, None, 4, 8, 1e-6, 0, None) == -1
    assert lib.dsw_rmsnorm_fwd(p, 8, None, 0, p, p, None, None, 4, 8, math.nan, 0, None) == -1
    assert lib.dsw_rmsnorm_fwd(p, 8, None, 0, p, p, None, None, 4, 0, 1e-6, 0, None) == -1
    assert lib.dsw_rmsnorm_fwd(None, 8, None, 0, None, None, None, None, 0, 8, 1e-6, 0, None) == 0   # no rows: nothing to do
    assert lib.dsw_rmsnorm_fwd_fp8(p, 8, None, 0, p, p, p, 3, None, 4, 8, 1e-6, 0, None) == -1       # scales overlap
    assert lib.dsw_quant_fp8(p, 8, None, p, 4, 4, 8, 0, None) == -1
    assert lib.dsw_quant_fp8_weight(p, 1, 8, p, None, 8, 8, 0, None) == -1
    need = lib.dsw_rmsnorm_bwd_workspace_bytes(1000, 256, 1)
    assert need > 0 and need % (256 * 4) == 0
    assert lib.dsw_rmsnorm_bwd_workspace_bytes(1000, 256, 3) == -2
    assert lib.dsw_rmsnorm_bwd(p, None, p, 256, None, 0, p, p, p, p, p, need - 1, 1000, 256, 1, None) == -3
    assert lib.dsw_rmsnorm_bwd(p, None, p, 256, None, 0, p, p, None, None, p, need, 1000, 256, 1, None) == -1
    assert lib.dsw_rmsnorm_bwd(p, None, p, 256, p, 255, p, p, p, p, p, need, 1000, 256, 1, None) == -1
    assert lib.dsw_fp8_mix_workspace_bytes(-1, 8, 8, 1) == -1
    assert lib.dsw_fp8_mix_workspace_bytes(1000, 8, 20, 1) == 0 and lib.dsw_fp8_mix_workspace_bytes(1000, 8, 20, 0) == 1008 * 32
    assert lib.dsw_fp8_mix(p, 20, p, 1, 1, p, 20, p, None, p, 1000, 8, 20, 0, p, 100, None) == -3
    assert lib.dsw_fp8_mix(p, 8, p, 1, 1, p, 7, p, None, p, 4, 8, 8, 0, None, 0, None) == -1
    assert lib.dsw_fp8_mix(p, 8, p, 1, 1, p, 8, p, None, p, 1 << 30, 1 << 8, 8, 0, p, 1 << 50, None) == -1      # 2^26 tiles
    assert lib.dsw_fp8_mix(p, 1 << 23, p, 1, 1, p, 8, p, None, p, 4, 8, 8, 0, None, 0, None) == -1
    assert lib.dsw_fp8_mix(p, 8, p, 1, 1, p, 8, p, None, p, 4, 8, 8, 5, None, 0, None) == -2
    assert lib.dsw_fp8_mix(None, 8, None, 1, 1, None, 8, None, None, None, 0, 8, 8, 0, None, 0, None) == 0
    assert b"overlap" in lib.dsw_strerror(-6)


def _clip(lib, ranges, outs=None, p=2.0, max_norm=1.0, ws=8192, dtypes=None, ws_bytes=None, norm=16):
    n = len(ranges)
    g = np.array([r[0] for r in ranges], dtype=np.uint64)
    o = np.array(outs if outs is not None else [r[0] for r in ranges], dtype=np.uint64)
    c = np.array([r[1] for r in ranges], dtype=np.int64)
    t = np.array(dtypes or [0] * n, dtype=np.int32)
    return lib.dsw_grad_norm_clip(n, g.ctypes.data, o.ctypes.data, c.ctypes.data, t.ctypes.data, p, max_norm, norm, ws,
                                  lib.dsw_grad_norm_workspace_bytes() if ws_bytes is None else ws_bytes, None)


def test_clip_entry_refuses_overlap_and_bad_arguments():
    lib = _native.load()
    assert _clip(lib, [(4096, 10), (4096, 10)]) == -6                        # one tensor listed twice
    assert _clip(lib, [(4096, 10), (4132, 10)]) == -6                        # the last element of one is the first of the next
    assert _clip(lib, [(4096, 10), (8192, 10)], outs=[65536, 65572]) == -6   # two outputs
    assert _clip(lib, [(4096, 10), (8192, 10)], outs=[8192, 65536]) == -6    # an output over another gradient
    assert _clip(lib, [(4096, 10)], outs=[4100]) == -6                       # an output shifted against its gradient
    assert _clip(lib, [(4096, 10), (4096, 0)], p=3.0) == -1
    assert _clip(lib, [(4096, 10)], max_norm=math.nan) == -1
    assert _clip(lib, [(4096, -1)]) == -1
    assert _clip(lib, [(0, 4)]) == -1
    assert _clip(lib, [(4096, 4)], dtypes=[9]) == -2
    assert _clip(lib, [(4096, 4)], ws_bytes=8) == -3
    assert _clip(lib, [(4096, 4)], ws=None) == -3
    assert _clip(lib, [(4096, 4)], norm=None) == -1
    assert lib.dsw_grad_norm_clip(-1, None, None, None, None, 2.0, 1.0, 16, 8192, 1 << 20, None) == -1


def test_rows_of_views():
    """(rows, stride) of the layouts the row kernels read in place, and the copies of the others."""
    as_rows = _native.ops().as_rows
    t = torch.arange(2 * 6 * 40, dtype=torch.float32).view(2, 6, 40)
    for view, rows, step in ((t, 12, 40), (t[..., 8:24], 12, 40), (t[1], 6, 40), (t[0, 0], 1, 40), (t[:, :1], 2, 240), (t[:1, 2:5, :7], 3, 40)):
        got = as_rows(view, False)
        assert got[0].data_ptr() == view.data_ptr() and got[1] == rows and (rows == 1 or got[2] == step), (view.shape, got[1:])
    for view in (t[:, 1:5, :8], t.transpose(1, 2), t[..., ::2], t[:1, :1].expand(2, 6, 40), t.flip(-1)):
        got, rows, step = as_rows(view, False)
        assert got.is_contiguous() and step == view.shape[-1] and torch.equal(got, view)
    scale = torch.empty(3, 12).view(3, 2, 6).movedim(0, -1)
    got, rows, step = as_rows(scale, True)
    assert got.data_ptr() == scale.data_ptr() and got.stride() == scale.stride() and (rows, step, got.stride(-1)) == (12, 1, 12)
    assert as_rows(torch.ones(1, 3).expand(12, 3), True)[2] == 0


def test_layers_and_bucket_reach_the_operators():
    from dsw_amd.parallel import FlatGradAllReduce, GradBucket
    from modules.layers import RMSNorm
    from modules.my_models_graph import _NodeLinear, serve_fp8

    norm = RMSNorm(8, eps=1e-5)
    assert [n for n, _ in norm.named_parameters()] == ["weight"] and bool((norm.weight == 1).all())
    with passed():
        norm(torch.randn(2, 3, 8))
    with passed():
        norm(torch.randn(2, 3, 8), torch.randn(2, 3, 8))
    with passed(), torch.no_grad():
        norm.rows_fp8(torch.randn(2, 3, 8))
    lin = _NodeLinear(8, 4)
    with passed():
        lin.serve_fp8()
    assert serve_fp8(torch.nn.Sequential(lin, torch.nn.ReLU()), enable=False) == 1
    for bucket in (GradBucket([lin.weight, lin.bias]), FlatGradAllReduce([lin.weight, lin.bias])):
        with passed():
            if not bucket.attached:
                lin.weight.grad = torch.ones_like(lin.weight)
            bucket.clip_norm(1.0)
    bucket = GradBucket([lin.weight, lin.bias])
    lin.weight.grad = None
    with pytest.raises(RuntimeError, match="no longer in the bucket"):
        bucket.clip_norm(1.0)
    with pytest.raises(ValueError, match="max_norm"):
        bucket.zero()
        bucket.clip_norm(-1.0)


def test_settling_collectives_waits_for_rccl_alone(monkeypatch):
    """Without a process group, or with gloo (whose calls are the host's), nothing waits; with RCCL the device is idle first."""
    from dsw_amd import parallel

    seen = []
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: seen.append("idle"))
    monkeypatch.setattr("time.sleep", lambda s: seen.append(s))
    parallel.settle_collectives()
    for backend, want in (("gloo", []), ("nccl", ["idle", 0.5])):
        seen.clear()
        monkeypatch.setattr(parallel.dist, "is_initialized", lambda: True)
        monkeypatch.setattr(parallel.dist, "get_backend", lambda *a, b=backend: b)
        parallel.settle_collectives()
        assert seen == want
