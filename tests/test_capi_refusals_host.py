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
