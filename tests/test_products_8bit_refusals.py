"""Products in 8-bit integers on the host: what the entry points refuse before anything is launched."""
import pytest

from fieldrun_b200.csrc import ops


@pytest.mark.parametrize("place", [1, 4, 8, 255])
def test_scratch_off_16_bytes_is_refused_before_any_kernel_writes_to_it(place):
    lib, room = ops.library("products8"), 1 << 40
    calls = {
        "linear": lambda: lib.frb_linear_8bit(None, 0, 9, 100, None, None, 33, None, 0, 0, place, room, None, None),
        "gated block": lambda: lib.frb_gated_8bit(None, 0, 3, 100, None, None, 40, None, None, 0, 0.0, None, 0, 0, place, room, None, None),
        "experts": lambda: lib.frb_expert_rows_8bit(None, 0, 3, 100, 1, None, None, None, None, None, 5, 8, None, None, 5, 40, None, None, 0.0, None, place, room, None,
                                                    None),
        "experts ": lambda: lib.frb_experts_8bit(None, 0, 3, 100, 2, None, None, None, None, 5, 40, None, None, 0.0, 8, None, 0, place, room, None, None),
    }
    for what, call in calls.items():
        assert call() == -1, what
        assert lib.frb_last_error().decode() == f"{what.strip()} in 8 bits: the scratch starts on 16 bytes"
