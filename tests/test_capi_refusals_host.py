"""What the ctypes wrappers refuse before anything of the library is called. The guards for devices are left out here, so no GPU is needed; that they
are there is tested on one."""
import pytest
import torch


@pytest.fixture()
def unreached(capi, monkeypatch):
    """The wrappers' module, where nothing may come as far as the library."""
    def lib():
        raise AssertionError("called")
    monkeypatch.setattr(capi, "lib", lib)
    monkeypatch.setattr(capi, "_check_operands", lambda *args, **kw: None)
    monkeypatch.setattr(capi, "_check_rows", lambda *args: None)
    monkeypatch.setattr(capi, "_check_int32", lambda *args: None)
    return capi


@pytest.mark.parametrize("shape", [(), (1, 1, 4), (1, 3, 64)])
def test_a_gate_is_a_row_or_rows(unreached, shape):
    """A gate of another number of dimensions was taken for one row of D elements, wherever it ends."""
    x = torch.zeros(3, 64, dtype=torch.bfloat16)
    with pytest.raises(unreached.FswError) as e:
        unreached.add_norm(x, x, torch.zeros(shape, dtype=torch.bfloat16))
    assert e.value.code == unreached.E_SHAPE


def rows(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype)


def int32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


SIXTEEN = [rows(5, 2, 16, 64)] * 2
EIGHT = [rows(5, 2, 16, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)] * 2 + [rows(5, 2, 16, dtype=torch.uint8).view(torch.float8_e8m0fnu)] * 2


@pytest.mark.parametrize("caches", [SIXTEEN, EIGHT])
def test_a_shared_prefix_has_pages(unreached, caches):
    """Without them the call was the plain decode's, whatever prefix_len said, or ended in an error of another kind."""
    with pytest.raises(unreached.FswError) as e:
        unreached.attn_shared(rows(3, 4, 64), caches, None, 40, int32(3, 2), int32(3), 32, 0.125)
    assert e.value.code == unreached.E_NULL


@pytest.mark.parametrize("caches", [SIXTEEN[:1], EIGHT[:3], EIGHT + EIGHT[:1]])
def test_caches_are_two_tensors_or_four(unreached, caches):
    q, kv, table, lengths = rows(3, 4, 64), rows(3, 2, 64), int32(3, 2), int32(3)
    append = lambda c: unreached.kv_append8(q, kv, kv, rows(9, 64, dtype=torch.float32), lengths, lengths, c)  # noqa: E731
    decode = lambda c: unreached.attn_decode8(q, c, table, lengths, 32, 0.125)  # noqa: E731
    calls = [append, decode, lambda c: unreached.kv_read(c, table, int32(4), 7, torch.bfloat16),
             lambda c: unreached.attn_shared(q, c, int32(3), 40, table, lengths, 32, 0.125)]
    for call in calls:
        with pytest.raises(unreached.FswError) as e:
            call(caches)
        assert e.value.code == unreached.E_SHAPE
    for call in calls[:2]:  # 8 bits alone
        with pytest.raises(unreached.FswError) as e:
            call(SIXTEEN)
        assert e.value.code == unreached.E_SHAPE
