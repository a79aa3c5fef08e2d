"""What the plan of attn_shared makes of the calls of test_shared_tiles_gpu.py: rows of a workgroup, tiles of 64 keys in a share, shares that a workgroup
takes in by itself or leaves to the join. A change of the plan that leaves a form of the kernels without its test fails here."""
import pytest

# sequences, query heads, key-value heads, channels, page size, prefix; rows of a workgroup; tiles of a share, at least
TILES = [
    (2, 128, 128, 64, 16, 1500, 64, 3), (3, 64, 64, 64, 64, 1000, 64, 2), (4, 16, 1, 48, 16, 20001, 64, 3),
    (2, 128, 128, 128, 16, 1500, 64, 3), (2, 128, 128, 80, 32, 1500, 64, 3),
    (2, 128, 128, 256, 16, 1500, 64, 3), (2, 64, 64, 192, 4, 1000, 64, 4),
    (99, 64, 1, 64, 16, 1500, 128, 5), (70, 8, 2, 64, 64, 9000, 128, 4), (40, 64, 1, 32, 16, 3000, 128, 4),
    (64, 32, 4, 128, 16, 2500, 128, 2), (128, 16, 2, 96, 8, 3000, 128, 3),
    (99, 64, 1, 128, 16, 9000, 256, 8),
    (32, 64, 4, 256, 16, 1500, 128, 3)]
# pages that the keys which a wave loads at a time do not fit: 64 rows, whatever the plan
ODD_TILES = [
    (2, 128, 128, 64, 5, 1500, 64, 3), (70, 8, 2, 64, 3, 9000, 64, 4), (99, 64, 1, 48, 12, 1500, 64, 5),
    (2, 128, 128, 128, 5, 1500, 64, 3), (40, 32, 1, 128, 3, 3000, 64, 3), (99, 64, 1, 112, 6, 1500, 64, 4),
    (2, 128, 128, 256, 3, 1500, 64, 3), (20, 64, 4, 256, 5, 1500, 64, 2)]
# of 8 bits alone: pages of 8 and of 24 tokens, loads of 16 keys
ODD_TILES_OF_8 = [(70, 8, 2, 64, 8, 9000, 64, 4), (2, 128, 128, 64, 24, 1500, 64, 3)]
# sequences, query heads, key-value heads, channels, page size, prefix, largest own length; shares of the prefix, at least; shares of own keys, at least. More
# shares of the prefix than 16 for each thread of a result, so that the join adds them whatever the own keys are.
JOINED = [
    (1, 8, 1, 64, 16, 20001, 60, 65, 1), (3, 8, 1, 64, 16, 9000, 900, 65, 4), (2, 16, 2, 64, 5, 4001, 60, 33, 1),
    (3, 8, 1, 128, 16, 3000, 900, 33, 4), (1, 8, 1, 128, 16, 20001, 40, 65, 1), (3, 16, 2, 112, 24, 2000, 900, 17, 2), (2, 8, 1, 128, 3, 5000, 50, 65, 1),
    (3, 8, 1, 256, 16, 3000, 900, 33, 4), (1, 8, 1, 256, 16, 30001, 50, 65, 1), (3, 8, 1, 208, 2, 2000, 700, 17, 2)]


def shares(capi, bits, B, Hq, Hkv, D, prefix, most):
    """Shares of the prefix, and of own keys up to `most`: a row of sums for each is what the scratch has."""
    L = capi.lib()
    size = L.fsw_attn_shared8_workspace_bytes if bits == 8 else L.fsw_attn_shared_workspace_bytes
    row = B * Hq * (D + 2) * 4
    none, own = (size(0, B, Hq, Hkv, D, prefix, n) for n in (0, most))
    assert none % row == own % row == 0
    return none // row - 1, (own - none) // row + 1


def rows_of(capi, bits, B, Hq, Hkv, D, page, prefix):
    L = capi.lib()
    return (L.fsw_attn_shared8_rows if bits == 8 else L.fsw_attn_shared_rows)(0, B, Hq, Hkv, D, prefix, page)


def check_tiles(capi, bits, B, Hq, Hkv, D, page, prefix, rows, least):
    assert rows_of(capi, bits, B, Hq, Hkv, D, page, prefix) == rows
    count, tiles = shares(capi, bits, B, Hq, Hkv, D, prefix, 0)[0], -(-prefix // 64)
    assert -(-tiles // count) >= least and prefix % 64 != 0, "%d tiles in %d shares" % (tiles, count)


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("case", TILES + ODD_TILES, ids=str)
def test_shares_of_several_tiles(capi, case, bits):
    check_tiles(capi, bits, *case)


@pytest.mark.parametrize("case", ODD_TILES_OF_8, ids=str)
def test_shares_of_several_tiles_of_8_bits(capi, case):
    check_tiles(capi, 8, *case)


def test_every_form_has_a_share_of_several_tiles():
    forms = {(max(64, 1 << (c[3] - 1).bit_length()), c[6]) for c in TILES}
    assert forms == {(64, 64), (64, 128), (128, 64), (128, 128), (128, 256), (256, 64), (256, 128)}
    assert {max(64, 1 << (c[3] - 1).bit_length()) for c in ODD_TILES} == {64, 128, 256}
    assert any(c[3] == 128 and c[6] == 256 for c in TILES)


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("case", JOINED, ids=str)
def test_shares_that_the_join_adds(capi, case, bits):
    B, Hq, Hkv, D, _, prefix, most, least, own = case
    results = Hq // Hkv * (16 if D <= 64 else 32 if D <= 128 else 64)     # four channels each; a workgroup has 256 threads
    count, own_shares = shares(capi, bits, B, Hq, Hkv, D, prefix, most)
    assert count >= least and count > 16 * max(1, 256 // results) and own_shares >= own and (own_shares == 1) == (own == 1)


def test_rows_of_what_is_refused_or_has_no_prefix(capi):
    for f, d in ((capi.lib().fsw_attn_shared_rows, 72), (capi.lib().fsw_attn_shared8_rows, 80)):
        assert f(0, 1, 8, 2, d, 100, 16) == 64
        for bad in ((2, 1, 8, 2, d, 100, 16), (0, 0, 8, 2, d, 100, 16), (0, 65536, 8, 2, d, 100, 16), (0, 1, 8, 3, d, 100, 16), (0, 1, 8, 2, d + 4, 100, 16),
                    (0, 1, 8, 2, d, 0, 16), (0, 1, 8, 2, d, (1 << 30) + 1, 16), (0, 1, 8, 2, d, 100, 0), (0, 1, 8, 2, d, 100, (1 << 30) + 1)):
            assert f(*bad) == 0, bad
    assert capi.lib().fsw_attn_shared8_rows(0, 1, 8, 2, 72, 100, 16) == 0
