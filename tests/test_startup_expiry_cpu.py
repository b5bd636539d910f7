"""A wait that expires in a start-up trial whose second try goes well drops no candidate, but its count has to be cleared all the
same: the chosen schedule was taken for unhealthy at the first check (three processes time-sharing one GPU)."""
import contextlib
import inspect
import time
from types import SimpleNamespace

import pytest
import torch
import torch.distributed as dist

from distributed_tensorflow_amd.parallel import dp_startup, schedule_select as sel
from test_schedule_select_cpu import US8, FakeOps, _run


def test_an_expiry_that_drops_nothing_is_reported():
    cands = ["ipc-shard", sel.REFERENCE]
    ops = FakeOps(US8, expire_once=[sel.REFERENCE])
    _, _, broken = _run(ops, cands, forced="ipc-shard")
    assert not broken and ops.expired_seen
    quiet = FakeOps(US8)
    _, _, broken = _run(quiet, cands, forced="ipc-shard")
    assert not broken and not quiet.expired_seen
    dropped = FakeOps(US8, expire=["ipc-shard"])
    _, _, broken = _run(dropped, cands)
    assert broken == {"ipc-shard"} and dropped.expired_seen


def test_the_start_up_clears_the_count_after_any_expiry():
    source = inspect.getsource(dp_startup)
    at = source.index("comm.reset_errors()")
    assert "if broken or ops.expired_seen:" in source[at - 400:at]


class _Exchange:
    """An exchange buffer that only counts: expired waits, resets, time-outs."""

    def __init__(self):
        self.errors, self.resets, self.timeouts = 0, 0, []

    def set_timeout(self, sec):
        self.timeouts.append(sec)

    def reset_errors(self):
        self.errors, self.resets = 0, self.resets + 1


class _Trainer(dp_startup.StartupMixin):
    """The start-up itself over an engine of four CPU tensors; the waits of ``expire``'s schedules run out in their first step."""

    def __init__(self, expire):
        self.rank, self.world, self.group, self._stage_host, self._shared_gpu = 0, 1, None, True, False
        self.ipc, self.ipc_act, self.ipc_w = _Exchange(), None, None
        self.startup_log, self.schedule, self.expire, self.steps, self._t_start = [], "", set(expire), 0, time.perf_counter()
        z = lambda: torch.zeros(8)  # noqa: E731
        self.engine = SimpleNamespace(P=z(), M=z(), V=z(), G=z(), step_t=torch.zeros(1), metrics_ring=z(), _steps_done=0, device="cpu", grad_hook=None,
                                      stream=SimpleNamespace(synchronize=lambda: None), bucket_bounds=lambda: [(0, 4), (4, 8)],
                                      fc1_grad_numel=lambda: 4)

    def prepare(self):
        pass

    def _ctx(self):
        return contextlib.nullcontext()

    def _use_schedule(self, name):
        self.schedule = name

    def transport_errors(self):
        return self.ipc.errors

    def materialize(self):
        pass

    def _wsh_reload(self):
        pass

    def train_steps(self, n):
        self.steps += n
        if self.schedule in self.expire:
            self.expire.discard(self.schedule)
            self.ipc.errors += 1
        else:
            self.engine.M += 0.1  # (a first moment of the gradient 1)


@pytest.mark.parametrize("expire,resets", [([], 0), ([sel.REFERENCE], 1), (["ipc-zerocopy"], 1)])
def test_the_chosen_schedule_starts_with_a_clean_count(expire, resets, monkeypatch):
    """Nothing expired: nothing is reset.  A first try that was repeated, or a candidate that was dropped: the count is zero again."""
    for k in ("DTF_DP_SCHEDULE", "DTF_DP_FAULT_INJECT", "DTF_DP_STARTUP_BUDGET_S", "DTF_IPC_FORCE_OVERLAP"):
        monkeypatch.delenv(k, raising=False)
    dist.init_process_group("gloo", store=dist.HashStore(), rank=0, world_size=1)
    try:
        t = _Trainer(expire)
        t._tune_schedule(allow_rccl=False, steps=16)
    finally:
        dist.destroy_process_group()
    assert t.ipc.errors == 0 and t.ipc.resets == resets and not t.expire
    assert t.schedule and t.schedule not in expire or expire == [sel.REFERENCE]
    assert t.steps > 16 and not t.engine.M.any() and t.engine._steps_done == 0  # trials ran, from the snapshot that is there again
    assert ("trying once more" in " ".join(t.startup_log)) == (expire == [sel.REFERENCE])
