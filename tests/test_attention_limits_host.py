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


def test_caches_whose_cells_overlap_are_not_written(capi):
    """Any order of the dimensions, but each inside the next larger stride; reading does not mind."""
    def append(strides, pages=4, page_size=16):
        return capi.lib().fsw_validate_kv_append(0, 4, 4, 2, 64, 64, P, 256, 64, P, 128, 64, P, 128, 64, P, 8, P, P, P, 256, 64,
                                                 P, 128, 64, cache_of(capi, pages, page_size, strides))
    for strides in ((2048, 1024, 64), (2048, 64, 128), (64, 4096, 256), (4096, 2048, 64), (2056, 1032, 64)):
        assert append(strides) == capi.OK, strides
    assert append((0, 1024, 64), pages=1) == append((128, 64, 0), page_size=1) == capi.OK
    assert append((1 << 40, 64, 128), pages=1 << 26) == append((64, 1 << 40, 1 << 24), page_size=1 << 16) == capi.OK
    for strides in ((64, 64, 64), (1024, 1024, 64), (2040, 1024, 64), (2048, 1032, 64), (2048, 960, 64), (2048, 64, 64), (2048, 64, 120), (64, 4096, 248),
                    (64, 1016, 256)):
        assert append(strides) == capi.E_LD, strides
        assert capi.lib().fsw_validate_attn_decode(0, 3, 4, 2, 64, P, 256, 64, cache_of(capi, strides=strides), P, 4, P, 64, 0.125, P, 256,
                                                   64) == capi.OK
    assert append((1 << 24, 64, 1 << 24), pages=1 << 26) == append((1 << 40, 1 << 40, 64), pages=1 << 26) == capi.E_LD


def test_rows_of_a_prompts_workgroup(capi):
    rows = capi.lib().fsw_attn_prompt_rows
    assert rows(0, 24, 1, 16, 4, 64) == rows(1, 2000, 1, 32, 8, 128) == 64
    assert rows(0, 8192, 1, 64, 8, 128) == rows(1, 1 << 20, 65535, 1024, 1024, 256) == 128
    assert rows(0, 0, 1, 4, 2, 64) == rows(2, 9, 1, 4, 2, 64) == rows(0, 9, 1, 4, 3, 64) == rows(0, 9, -1, 4, 2, 64) == rows(0, 9, 1, 4, 2, 12) == 0


def test_shares_of_few_items(capi):
    """Between 128 and 256 items too few workgroups would run on an unsplit bound: their keys are shared by two."""
    ws = capi.lib().fsw_attn_decode_workspace_bytes
    for B in (15, 16, 20, 31):
        assert ws(0, B, 64, 8, 128, 2300) > 0, B
    assert ws(0, 32, 64, 8, 128, 2300) == ws(0, 64, 64, 8, 128, 2300) == ws(0, 16, 64, 8, 128, 512) == 0
