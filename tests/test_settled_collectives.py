"""Before RCCL collectives are recorded the process group's watchdog has nothing left to ask for: waited for, not hoped for."""
import torch

from dsw_amd import parallel


def test_every_rccl_group_is_drained_behind_an_idle_device(monkeypatch):
    class Group:
        def __init__(self, name, backend):
            self.name, self.backend = name, backend

        def _wait_for_pending_works(self):
            seen.append(self.name)

    seen = []
    groups = {Group("world", "nccl"): None, Group("host", "gloo"): None, Group("pair", "nccl"): None}
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: seen.append("idle"))
    monkeypatch.setattr("time.sleep", lambda s: None)
    monkeypatch.setattr(parallel.dist, "is_initialized", lambda: True)
    monkeypatch.setattr(parallel.dist, "get_backend", lambda group=None: "nccl" if group is None else group.backend)
    monkeypatch.setattr(parallel, "_process_groups", lambda: list(groups), raising=False)
    parallel.settle_collectives()
    assert seen == ["idle", "world", "pair"]


def test_the_groups_of_a_real_world_can_be_drained(tmp_path):
    import torch.distributed as dist

    dist.init_process_group("gloo", rank=0, world_size=1, init_method="file://%s" % (tmp_path / "store"))
    try:
        other = dist.new_group([0])
        found = parallel._process_groups()
        assert any(g is dist.group.WORLD for g in found) and any(g is other for g in found)
        assert all(callable(g._wait_for_pending_works) for g in found)
        parallel.settle_collectives()                 # gloo: nothing to wait for
    finally:
        dist.destroy_process_group()
    assert parallel._process_groups() == []
