"""Limits of the chunk entry points, before any launch: no GPU needed."""

import pytest

import branchcraft_capi as capi

FAKE = 0x1000  # a non-null address; never dereferenced on the rejection path


@pytest.mark.parametrize("batch", [(1 << 24) - 1, 1 << 24, (1 << 31) - 1])
def test_build_tables_rejects_more_requests_than_a_launch_takes(batch):
    args = [FAKE, 9, FAKE, FAKE, batch, 4, 3, FAKE, FAKE, FAKE, FAKE, None]
    assert capi.load().bc_build_tables(*args) == capi.BC_ERROR_INVALID_VALUE
