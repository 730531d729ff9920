"""Refusals of the paged 4-bit cache's C entries that need no device."""
import pytest

from gemma_triton_flash_attn import _lib

FAKE = 0x100000  # never dereferenced: validation fails first


@pytest.mark.parametrize("D,N,B,H", [(64, 2 ** 31 - 1, 1, 1), (64, 2 ** 31 - 127, 1, 1), (512, 2 ** 28, 1, 1),
                                     (64, 1, 65536, 1), (64, 1, 1, 65536)])
def test_append_refuses_sizes_whose_indices_pass_32_bits(D, N, B, H):
    """The last CTA's (token, group) pairs run past the last token: beyond 2^31 - 128 groups they would come back
    as negative tokens. Refused before a device is looked for."""
    st = _lib.strides_arg((8, 8, 8, 1))
    rc = _lib.load().gqafa_kv4_append(FAKE, st, FAKE, st, FAKE, 0, FAKE, 9, B, H, N, D, 64, 1, None)
    assert rc == _lib.GQAFA_ERR_INVALID and b"out of range" in _lib.load().gqafa_last_error()
