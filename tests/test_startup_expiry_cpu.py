"""A wait that expires in a start-up trial whose second try goes well drops no candidate, but its count has to be cleared all the
same: the chosen schedule was taken for unhealthy at the first check (three processes time-sharing one GPU)."""
import inspect

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
