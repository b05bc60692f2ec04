"""laic_dev_wait_stream without a GPU."""


def test_null_engine_is_refused():
    from laicompute_b200._native import LAIC_E_INVALID, lib
    assert lib().laic_dev_wait_stream(None, None) == LAIC_E_INVALID
    assert b"null device" in lib().laic_last_error()
