"""What the paged cache's entry points answer without a device."""
import ctypes as C

import pytest

from tuckmill_b200 import cuda


def test_shapes_that_pages_serve():
    for hd in (0, 16, 32, 48, 64, 96, 128, 192, 256, 512):
        for page in (0, 1, 8, 16, 24, 32, 64, 128, 256, 512):
            assert cuda.kv_pages_supported(hd, page) == (hd in (32, 64, 128, 256) and page in (16, 32, 64, 128, 256))


def test_scratch_grows_with_counted_rows_only():
    plain = cuda.attention_paged_scratch_bytes(4, 16, 8, 128, 64, 100)
    assert plain == cuda.attention_paged_scratch_bytes(900, 64, 8, 128, 16, 7) > 0  # what CTAs leave behind
    counted = cuda.attention_paged_scratch_bytes(4, 16, 8, 128, 64, 100, True)
    assert counted == plain + 4 * 16 * 4 * (2 + 6400)  # a score a row and head, a maximum and a sum a head
    assert cuda.attention_paged_scratch_bytes(1024, 1024, 32, 256, 256, 1 << 17, True) > 1 << 47  # no 32-bit product


@pytest.mark.parametrize("name,args", [
    ("attention_decode_paged_dev", [None] * 16 + [1] * 11 + [1.0, 1.0]),
    ("kv_pages_copy_f16", [None] * 6 + [1] * 6 + [1, 1, None]),
    ("kv_pages_evict", [None] * 10 + [1] * 9),
    ("logits_adjust_rows_f32_dev", [None, None, 1, 1, None, 1, 0, None, 1] + [None] * 5 + [0, None, None, None]),
])
def test_no_context_is_refused(name, args):
    err = C.create_string_buffer(128)
    assert getattr(cuda.load_library(), "tm_cuda_" + name)(None, *args, err, 128) == -5
    assert b"context" in err.value
