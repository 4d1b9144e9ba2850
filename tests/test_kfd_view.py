"""The GPU tests that need KFD's view of each process are skipped, and said to be, only where there is none."""

import ast
from pathlib import Path
from types import SimpleNamespace

import conftest
import pytest


class Item(SimpleNamespace):
    def add_marker(self, mark):
        self.marks.append(mark)


def items():
    out = [Item(originalname=n, path=Path(f), marks=[]) for f, names in conftest.NEEDS_KFD_PROC.items() for n in names]
    return out, [Item(originalname="test_queue_cap_protects_masked_neighbours", path=Path("test_shim_interpose_gpu.py"), marks=[]),
                 Item(originalname="test_attention", path=Path("test_paged_ops_gpu.py"), marks=[])]


@pytest.mark.parametrize("there", [True, False])
def test_skipped_only_without_the_view(tmp_path, monkeypatch, there):
    if there:
        (tmp_path / "proc").mkdir()
    monkeypatch.setattr(conftest, "KFD_PROC", tmp_path / "proc")
    listed, others = items()
    conftest.pytest_collection_modifyitems(listed + others)
    assert all(not i.marks for i in others)
    for i in listed:
        assert [m.name for m in i.marks] == ([] if there else ["skip"])
        assert there or "KFD" in i.marks[0].kwargs["reason"]


def test_every_listed_test_is_there_and_a_gpu_test():
    for name, tests in conftest.NEEDS_KFD_PROC.items():
        tree = ast.parse((Path(__file__).parent / name).read_text())
        assert tests <= {f.name for f in tree.body if isinstance(f, ast.FunctionDef)}, name
        assert "pytest.mark.gpu" in ast.unparse(tree), name
