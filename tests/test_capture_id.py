"""kv800_hip_capture_id's host checks (CPU)."""
import lfm3_kv800_amd.kv800_hip as kh


def test_a_null_pointer_is_refused():
    L = kh.load_library()
    assert L.kv800_hip_capture_id(None, None) == -1 and b"capture_id" in L.kv800_hip_last_error()
