"""More of the operators over many sequences, beside tests/test_sequences_gpu.py: sizes that wrap."""
import numpy as np
import pytest

from sharpinference_amd import native

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("size,slots", [(1 << 36, 1 << 28), ((1 << 36) - 4096, (1 << 31) - 1), (1 << 35, (1 << 29) + 1),
                                        (1 << 33, (1 << 31) - 1)])
def test_copy_slots_beyond_the_address_space(hip, size, slots):
    """slots * slot_bytes at 2^64 and beyond (modulo that, these arrays would be small or lie anywhere): refused."""
    b = hip.alloc(1 << 16)
    pair = [hip.to_device(np.full(1, -1, np.int32)) for _ in range(2)]
    with pytest.raises(native.HipError) as e:
        hip.copy_slots(native.slot_arrays([(b.ptr, size)]), slots, pair[0].ptr, pair[1].ptr, 1)
    assert e.value.status == native.ERR_ARGUMENT
    for x in [b, *pair]:
        x.free()
