"""What the paged cache's entry points answer without a device."""
import ctypes as C

import pytest

from tuckmill_b200 import cuda


def test_shapes_that_pages_serve():
    for hd in (0, 16, 32, 48, 64, 96, 128, 192, 256, 512):
        for page in (0, 1, 8, 16, 24, 32, 64, 128, 256, 512):
            assert cuda.kv_pages_supported(hd, page) == (hd in (32, 64, 128, 256) and page in (16, 32, 64, 128, 256))


def test_scratch_of_a_call():
    plain = cuda.attention_paged_scratch_bytes(4, 16, 8, 128, 64, 100)
    assert plain == cuda.attention_paged_scratch_bytes(4, 16, 8, 128, 16, 7) > 0  # without weights the cache's length is no matter
    counted = cuda.attention_paged_scratch_bytes(4, 16, 8, 128, 64, 100, True)
    assert counted == plain + 4 * 16 * 4 * 6400  # a score a row and head
    assert cuda.attention_paged_scratch_bytes(1024, 1024, 32, 256, 256, 1 << 17, True) > 1 << 47  # no 32-bit product
    for heads, kvh, hd, page in ((3, 2, 64, 16), (4, 0, 64, 16), (4, 2, 48, 16), (4, 2, 64, 24)):
        assert cuda.attention_paged_scratch_bytes(1, heads, kvh, hd, page, 4) == 0


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


@pytest.mark.parametrize("runs", [[(0, 0, 5)], [(0, 0, 0, 5), (1, 1)], [(0, 0, 0), (5, 1, 1, 0, 2)], [(), (0, 0, 0, 5, 1, 1, 0, 2)]])
def test_runs_of_a_page_copy_are_four_numbers_each(runs):
    with pytest.raises(ValueError):
        cuda.CudaContext.kv_pages_copy(None, None, None, None, None, None, None, 1, 16, 1, 1, 64, 16, True, runs)
