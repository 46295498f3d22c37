"""What attention over trees refuses beside tests/test_drafts_host.py (no GPU: tensors without memory stand in)."""

import pytest

from tests.test_drafts_host import KernelError, attend, device_zero, fake  # noqa: F401  (the fixture)


@pytest.mark.parametrize("change,why", [
    ({"window": 1 << 31, "positions": lambda: fake(6)}, "below 2\\^31"),
    ({"window": 1 << 40, "positions": lambda: fake(6)}, "below 2\\^31"),
    ({"max_context": 1 << 31}, "below 2\\^31"),
])
def test_numbers_that_do_not_fit_are_refused(change, why):
    """(an int of the entry point takes 32 bits: a window of 2^40 would have been none at all)"""
    with pytest.raises(KernelError, match=why):
        attend(**change)
