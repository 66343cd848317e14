"""CPU checks of what the generation entries and their Python wrappers do before any launch."""
import pytest


@pytest.fixture(scope="module")
def lib():
    from decisive_b200 import build, _lib
    build.build()
    return _lib.load()


ONE = 4 * 128 * 128  # floats of a state of 4 heads


# Addresses in floats from a base that no device tensor has: every call is refused before it could launch anything.
@pytest.mark.parametrize("items,state,stride,state_out", [
    (3, 2 * ONE, 0, 0),         # a kept state that is a slot of the output
    (3, 0, 0, 0),               # ... the first one
    (2, ONE - 4, 0, 0),         # ... that ends inside
    (2, 0, 0, ONE - 4),         # ... that the output begins in
    (3, 0, ONE, ONE),           # states moved up by one item
    (3, ONE, ONE, 0),           # ... and down
    (2, 0, 2 * ONE, 0),         # every other state, packed
    (3, 0, 4 * ONE, 6 * ONE),   # the output lies over the third state of a wide stride
    (1, 0, ONE, 4), (1, 4, 0, 0),
])
def test_delta_refuses_states_that_meet(lib, items, state, stride, state_out):
    base = 1 << 20
    rc = lib.db_gated_delta(16, 16, 16, 1, 512, 512, 512, 16, 16, 4, 4, None, items, 4 * items, 4, 2, 4, 128, 1.0, -1.0,
                            base + 4 * state, stride, base + 4 * state_out, 16, 512, None, None)
    assert rc == -1 and lib.db_last_error_code() == b"INVALID_ARGUMENT"
