"""The paged cache's C entry points without a GPU: null arguments are errors."""
import focr_hip


def test_null_arguments_are_errors_not_crashes():
    lib = focr_hip.lib()
    assert lib.focr_kv_pages_create(None, 4, 16, 1, 4, 16, 8, 8, 64, None) == -1
    assert "null" in lib.focr_last_error().decode()
    assert lib.focr_kv_pages_map(None, None, 0, 0, 0, None) == -1
    assert lib.focr_kv_pages_append(None, None, None, None, 1, None, None, 1) == -1
    assert lib.focr_kv_pages_qkv_rows(None, None, None, 1, None, None, None, 1, None) == -1
    assert lib.focr_kv_pages_attention(None, None, None, 1, None, None, 1, 1, None, None) == -1
    assert lib.focr_kv_pages_dequantize(None, None, 1, None, None, 1, None, None) == -1
    assert lib.focr_kv_pages_refused(None, None, None) == -1
    assert lib.focr_kv_pages_info(None, None, None, None, None, None) == -1
    assert lib.focr_kv_pages_free(None) == 0
