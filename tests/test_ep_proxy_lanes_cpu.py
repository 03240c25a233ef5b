"""How many streams the EP proxy's copy lanes share: the null stream and one
more of the application's keep hardware queues of their own."""

import pytest

import uccl_amd

if not uccl_amd.native_available():
    pytest.skip("native extension not built", allow_module_level=True)


@pytest.mark.parametrize("queues, streams", [
    (None, 2), ("4", 2), ("8", 6), ("32", 30), ("3", 1), ("2", 1), ("1", 1)])
def test_lanes_leave_two_queues(monkeypatch, queues, streams):
    if queues is None:
        monkeypatch.delenv("GPU_MAX_HW_QUEUES", raising=False)
    else:
        monkeypatch.setenv("GPU_MAX_HW_QUEUES", queues)
    assert uccl_amd._load_native(required=True).ep_proxy_lane_streams() == \
        streams
