"""A write or an import that is refused leaves the handle that it was to replace as it was."""
import pytest
import torch

import neuzip
from tests.fakes import cpu_manager
from tests.test_mx4_calls import blob_of
from tests.test_mx4_host import manager_with


def test_a_refused_write_leaves_the_handle_readable():
    m = cpu_manager(7)
    w = torch.arange(12, dtype=torch.bfloat16).reshape(3, 4)
    h = m.write(w)
    with pytest.raises(RuntimeError, match="Unsupported data type"):
        m.write(torch.zeros(5, 7), h)
    assert m.meta_dict[h] == (3, 4) and torch.equal(m.read(h), w)
    assert m.write(w.t().contiguous(), h) == h and m.read(h).shape == (4, 3)
    blob = m.export_entry(h)
    with pytest.raises(AssertionError):
        m.import_entry({**blob, "precision": 3, "shape": (12,)}, h)
    assert m.read(h).shape == (4, 3)


def test_a_refused_import_leaves_a_4_bit_handle_as_it_was():
    m = manager_with((32, 64))
    for change in ({"format": "NZR1"}, {"dtype": "float32"}, {"stack": (1, 4, 65)}, {"packed": torch.zeros(3)}):
        with pytest.raises(ValueError):
            m.import_entry({**blob_of((4, 64)), **change}, "w")
        assert m.meta_dict["w"] == (32, 64)
    with pytest.raises(RuntimeError, match="Unsupported data type"):
        m.write(torch.zeros(4, 64), "w")
    assert m.meta_dict["w"] == (32, 64)


def test_a_refused_new_handle_does_not_free_its_number():
    # another thread may have taken the next one meanwhile
    m = cpu_manager(7)
    with pytest.raises(RuntimeError):
        m.write(torch.zeros(2))
    assert m.write(torch.zeros(2, dtype=torch.bfloat16)) == "1"
    assert neuzip.Manager.total_size(m) == m.size("1")
