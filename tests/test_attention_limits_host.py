"""What the attention entry points accept and refuse at their limits, on the host."""
import ctypes

P = 0x1000  # a pointer that is never followed


def cache_of(capi, pages=4, page_size=16, strides=(2048, 1024, 64)):
    return ctypes.byref(capi.KvCache(P, P, pages, page_size, *strides))


def decode(capi, B=3, ld=4, max_len=64, scale=0.125):
    return capi.lib().fsw_validate_attn_decode(0, B, 4, 2, 64, P, 256, 64, cache_of(capi), P, ld, P, max_len, scale, P, 256, 64)


def test_one_row_of_pages_for_all_sequences(capi):
    assert decode(capi) == decode(capi, ld=0) == capi.OK
    assert decode(capi, ld=3) == decode(capi, ld=-1) == decode(capi, B=1, ld=0) == capi.E_LD


def prompt(capi, scale):
    return capi.lib().fsw_validate_attn_prompt(0, 9, 9, 2, 4, 2, 64, P, 256, 64, P, 128, 64, P, 128, 64, P, P, scale, P, 256, 64)


def test_scales_that_are_finite_times_log2_e(capi):
    """Scores are exponents of two: they are multiplied by scale log2(e), and a score of zero has to stay zero."""
    for scale in (2.0 ** -126, 1.0, 2.3e38):
        assert decode(capi, scale=scale) == prompt(capi, scale) == capi.OK
    for scale in (2.4e38, 3.4e38, float("inf"), float("nan"), 2.0 ** -127, 0.0, -1.0):
        assert decode(capi, scale=scale) == prompt(capi, scale) == capi.E_SHAPE
