"""CPU: when the comparisons with the reference project's own kernels are skipped, and when they are not."""
import pathlib

import pytest

from oracle import build_oracle
from tests import conftest


class Item:
    def __init__(self, name):
        self.path, self.marks = pathlib.Path("tests") / name, []

    def add_marker(self, mark):
        self.marks.append(mark)


@pytest.mark.parametrize("library", [False, True])
@pytest.mark.parametrize("checkout", [False, True])
def test_reference_comparisons_are_skipped_only_without_a_checkout(tmp_path, monkeypatch, library, checkout):
    monkeypatch.setattr(build_oracle, "REF_LIB", str(tmp_path / "lib.so"))
    monkeypatch.setattr(build_oracle, "DEFAULT_REFERENCE", str(tmp_path / "reference"))
    if library:
        (tmp_path / "lib.so").touch()
    if checkout:
        (tmp_path / "reference" / "src" / "impl").mkdir(parents=True)
    items = [Item("test_reference_gpu.py"), Item("test_gemm_gpu.py")]
    conftest.pytest_collection_modifyitems(None, items)
    assert [m.name for m in items[0].marks] == ([] if library or checkout else ["skip"])
    assert items[1].marks == []
